"""GPU: dense layers and the loss on top of one in each of their forms, whole outputs against 64 bits on the device.

What is compared is the norm of an output's error.  A sum of K products in fp32 whose partial sums grow as a random walk's is off by 0.41 sqrt(K) U of its own size (each addition by U / sqrt(3) of the
partial sum), and what is in front of it (halves, an activation's slope, a bias) by a few U: (sqrt(K) + 16) U, which a product without the lower halves of an operand, 2^-12, is far beyond."""
import math

import numpy as np
import pytest

import dense_sizes
from dense_reference import U

pytestmark = pytest.mark.gpu

ACTIVATIONS = ["none", "relu", "sigmoid", "hard_tanh"]


def generator(seed):
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return gen


def frames_of(gen, n, frames, pitch):
    """NaN behind the last frame"""
    import torch
    t = torch.full((n, pitch), math.nan, device="cuda")
    t[:, :frames] = torch.randn((n, frames), generator=gen, device="cuda")
    return t


def inputs_of(gen, n, frames, bit):
    """-> (x, its values in 64 bits)"""
    import torch
    if not bit:
        x = frames_of(gen, n, frames, frames + 3)
        return x, x[:, :frames].double()
    x = torch.randint(-(1 << 31), 1 << 31, (n, frames // 32 + 2), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32)
    at = torch.arange(frames, device="cuda")
    return x, ((x[:, at // 32] >> (at % 32).to(torch.int32)) & 1).double()


def activated(z, activation):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "sigmoid": lambda: z.sigmoid(), "hard_tanh": lambda: z.clamp(-1, 1)}[activation]()


def slope(y, activation):
    import torch
    return {"none": lambda: torch.ones_like(y), "relu": lambda: (y > 0).double(), "sigmoid": lambda: y * (1 - y), "hard_tanh": lambda: (y.abs() < 1).double()}[activation]()


def near(name, got, want, tolerance):
    import torch
    error = float(torch.linalg.norm(got.double() - want) / torch.linalg.norm(want))
    assert error <= tolerance, (name, error, tolerance)


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", list(dense_sizes.FORWARD))
def test_forward(size, bit):
    import torch
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    for k, activation in enumerate(ACTIVATIONS):
        gen = generator(k)
        x, values = inputs_of(gen, inputs, frames, bit)
        W = torch.randn((outputs, inputs), generator=gen, device="cuda") / math.sqrt(inputs)
        b = torch.randn(outputs, generator=gen, device="cuda")
        r = frames_of(gen, outputs, frames, frames + 1) if k % 2 else None
        if bit:
            y = ops.bit_dense_affine_forward(x, W, b, frames, frames + 2, activation=activation, residual=r)
        else:
            y = ops.dense_affine_forward(x, W, b, frames, activation=activation, residual=r)
        z = W.double() @ values + b.double()[:, None]
        if r is not None:
            z = z + r[:, :frames].double()
        near(activation, y[:, :frames], activated(z, activation), (math.sqrt(inputs) + 16) * U)


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", list(dense_sizes.BACKWARD))
def test_backward(size, bit):
    """dx, dW, db and dr through each activation, added to what is there or not"""
    import torch
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    call = ops.bit_dense_affine_backward if bit else ops.dense_affine_backward
    for k, activation in enumerate(ACTIVATIONS):
        gen = generator(10 + k)
        x, values = inputs_of(gen, inputs, frames, bit)
        W = torch.randn((outputs, inputs), generator=gen, device="cuda") / math.sqrt(inputs)
        dy = frames_of(gen, outputs, frames, frames + 5)
        y = None if activation == "none" else activated(frames_of(gen, outputs, frames, frames + 5), activation)
        given = {}
        if k % 2:
            given = dict(dW=torch.randn(W.shape, generator=gen, device="cuda"), db=torch.randn(outputs, generator=gen, device="cuda"))
        dW0, db0 = (given["dW"].double(), given["db"].double()) if given else (0.0, 0.0)
        dx, dW, db, dr = call(x, dy, W, frames, activation=activation, y=y, want_dr=True, **given)
        dz = dy[:, :frames].double()
        if y is not None:
            dz = dz * slope(y[:, :frames].double(), activation)
        near(activation + " dr", dr[:, :frames], dz, 4 * U)
        near(activation + " dx", dx[:, :frames], W.double().t() @ dz, (math.sqrt(outputs) + 16) * U)
        near(activation + " dW", dW, dz @ values.t() + dW0, (math.sqrt(frames) + 16) * U)
        near(activation + " db", db, dz.sum(1) + db0, (math.sqrt(frames) + 16) * U)


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", list(dense_sizes.LOSS))
def test_loss(size, bit):
    """labels in every piece, frames that do not count, gradients added to what is there.  A logit off by e moves a probability by 2 e at most; e is (sqrt(inputs) + 16) U of four times the logits' root
    mean square, which few exceed"""
    import torch
    from binarybrain_amd import ops
    inputs, channels, frames = size
    gen = generator(30)
    x, values = inputs_of(gen, inputs, frames, bit)
    W = torch.randn((channels, inputs), generator=gen, device="cuda") * (2.0 / math.sqrt(inputs))
    b = torch.randn(channels, generator=gen, device="cuda")
    label = torch.randint(0, channels, (frames,), generator=gen, device="cuda", dtype=torch.int32)
    weight = torch.rand(frames, generator=gen, device="cuda") + 0.5
    label[1::5], label[2::11], weight[::7] = -1, channels, 0.0
    counts = (label >= 0) & (label < channels) & (weight != 0)
    if not bit:
        x[:, :frames][:, ~counts] = math.nan
    values = torch.where(counts, values, 0.0)
    w = torch.where(counts, weight.double(), 0.0)
    weight_sum = float(w.sum())
    there = dict(dW=torch.randn(W.shape, generator=gen, device="cuda") / 100, db=torch.randn(channels, generator=gen, device="cuda") / 100)
    dW0, db0 = there["dW"].double(), there["db"].double()
    give = dict(weight=weight, weight_sum=weight_sum)
    call = (lambda **k: ops.bit_loss_dense_softmax_cross_entropy(x, W, b, label, frames, frames + 2, **give, **k)) if bit else \
           (lambda **k: ops.loss_dense_softmax_cross_entropy(x, W, b, label, frames, **give, **k))
    loss, dx, dW, db = call(**there)

    z = torch.addmm(b.double()[:, None], W.double(), values)
    off = 2 * (math.sqrt(inputs) + 16) * U * 4 * float(z.square().mean().sqrt())
    at, here = torch.where(counts, label, 0).long(), torch.arange(frames, device="cuda")
    top = z.amax(0)
    log_sum = (z - top).exp_().sum(0).log() + top
    want = torch.where(counts, w * (log_sum - z[at, here]), 0.0)
    z -= log_sum
    z.exp_()
    z[at, here] -= 1.0
    z *= torch.where(counts, w / weight_sum, 0.0)
    near("loss", loss[0, :frames], want, off + 16 * U)
    near("dx", dx[:, :frames], W.double().t() @ z, off + (math.sqrt(channels) + 16) * U)
    near("dW", dW - dW0, z @ values.t(), off + (math.sqrt(frames) + 16) * U + 2 * U * float(torch.linalg.norm(dW0) / torch.linalg.norm(z @ values.t())))
    near("db", db - db0, z.sum(1), off + (math.sqrt(frames) + 16) * U + 2 * U * float(torch.linalg.norm(db0) / torch.linalg.norm(z.sum(1))))
    assert not dx[:, :frames][:, ~counts].any() and not loss[0, :frames][~counts].any()
    # the loss alone has the same bits
    assert torch.equal(call(want_gradients=False)[0][0, :frames], loss[0, :frames])
