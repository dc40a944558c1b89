"""GPU: large dense products hold their operands to fp32's relative accuracy whatever else is in the row: values far below the largest of a row count as much as fp32 lets them, where the other
operand is as much larger there, or 0 where this one is large."""
import numpy as np
import pytest

import test_gpu_dense as cases
from dense_reference import U, bits_of, loss as exact_loss, through
from test_gpu_dense import dev, host, near, rows

pytestmark = pytest.mark.gpu

F32 = np.float32


def even_bound(a, b):
    """3 K roundings of a sum of K products (three products of halves each), 16 U for the halves themselves, and 2^-20 of a sum on its way, which is at most the sum of magnitudes, for what an element
    that is not formed again may have lost: nothing that goes by the largest value of a row"""
    k = a.shape[1]
    return ((3 * k + 16) * U + 2.0 ** -20) * (np.abs(a) @ np.abs(b))


def wide(rng, *shape, octaves=60):
    """magnitudes spread evenly over 2^-octaves .. 1"""
    return (rng.choice([-1.0, 1.0], shape) * 2.0 ** -rng.uniform(0, octaves, shape)).astype(F32)


# (inputs, outputs, frames): tiles of each size, whole and with a shared k axis (1103 inputs), long k axes
SIZES = [(300, 2600, 2500), (1103, 640, 1300), (145, 21806, 548), (4100, 1030, 1030), (640, 530, 1100)]


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_each_weight_alone(size, bit):
    """one input per frame is not 0: the output is that weight times it"""
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    rng = np.random.default_rng(1)
    W = wide(rng, outputs, inputs)
    at = rng.integers(0, inputs, frames)
    if bit:
        words = np.zeros((inputs, (frames + 31) // 32), np.uint32)
        np.bitwise_or.at(words, (at, np.arange(frames) // 32), np.uint32(1) << (np.arange(frames) % 32).astype(np.uint32))
        got, value = host(ops.bit_dense_affine_forward(dev(words.view(np.int32)), dev(W), None, frames, frames)), np.ones(frames)
    else:
        x = np.zeros((inputs, frames), F32)
        x[at, np.arange(frames)] = value = wide(rng, frames)
        got = host(ops.dense_affine_forward(dev(x), dev(W), None, frames))
    want = W.astype(np.float64)[:, at] * value
    assert np.all(np.abs(got - want) <= (16 * U + 2.0 ** -20) * np.abs(want))


@pytest.mark.parametrize("octaves", [10, 20, 25, 30])
@pytest.mark.parametrize("size", SIZES)
def test_inputs_of_other_scales(size, octaves):
    """eight inputs that much larger than the others, with weights as much smaller: all count alike"""
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    rng, x, values, W, b = cases.layer(2, inputs, outputs, frames, False, frames)
    at = rng.choice(inputs, 8, replace=False)
    x[at] *= F32(2.0 ** octaves)
    W[:, at] *= F32(2.0 ** -octaves)
    got = host(ops.dense_affine_forward(dev(x), dev(W), None, frames)).astype(np.float64)
    W64, x64 = W.astype(np.float64), x.astype(np.float64)
    want = W64 @ x64
    near(got, want, even_bound(W64, x64), "y")
    assert np.linalg.norm(got - want) <= 2.0 ** -20 * np.linalg.norm(want)


BACKWARD = [(300, 2600, 1100), (1024, 1001, 1000), (640, 530, 1100), (2048, 4300, 1500), (512, 700, 4200)]


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", BACKWARD)
def test_gradients_of_frames_of_any_scale(size, bit):
    """every third frame has gradients 2^35 times larger, and no input that is not 0: dW is of the others"""
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    rng, x, values, W, b = cases.layer(3, inputs, outputs, frames, bit, (frames + 31) // 32 * 32)
    dy = rows(rng, outputs, frames, frames)
    dy[:, ::3] *= F32(2.0 ** 35)
    y = rows(rng, outputs, frames, frames)
    if bit:
        on = np.ascontiguousarray(bits_of(x, frames).astype(np.uint8))
        on[:, ::3] = 0
        x = np.packbits(np.pad(on, ((0, 0), (0, -frames % 32))), axis=1, bitorder="little").view(np.int32)
        values = on.astype(np.float64)
    else:
        x[:, ::3] = 0.0
        values = x[:, :frames].astype(np.float64)
    call = ops.bit_dense_affine_backward if bit else ops.dense_affine_backward
    dx, dW, db, dr = call(dev(x), dev(dy), dev(W), frames, activation="relu", y=dev(y))
    dz = through(dy.astype(np.float64), y.astype(np.float64), "relu")
    near(host(dW), dz @ values.T, even_bound(dz, values.T), "dW")


@pytest.mark.parametrize("activation", ["none", "sigmoid"])
@pytest.mark.parametrize("size", BACKWARD)
def test_gradients_of_outputs_of_any_scale(size, activation):
    """every fifth output has gradients 2^32 times larger, and weights as much smaller; and each third output's weights are 0"""
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    rng, x, values, W, b = cases.layer(4, inputs, outputs, frames, False, frames)
    dy = rows(rng, outputs, frames, frames)
    dy[::5] *= F32(2.0 ** 32)
    W[::5] *= F32(2.0 ** -32)
    W[1::3] = 0.0
    dy[1::3] *= F32(2.0 ** 40)
    y = 1.0 / (1.0 + np.exp(-rows(rng, outputs, frames, frames)))
    dx = ops.dense_affine_backward(dev(x), dev(dy), dev(W), frames, activation=activation, y=None if activation == "none" else dev(y.astype(F32)), want_weights=False)[0]
    dz = through(dy.astype(np.float64), y.astype(F32).astype(np.float64), activation)
    W64 = W.astype(np.float64)
    near(host(dx)[:, :frames], W64.T @ dz, even_bound(W64.T, dz) + 4 * U * (np.abs(W64.T) @ np.abs(dz)), "dx")


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("confidence", [0.0, 12.0, 25.0])
@pytest.mark.parametrize("size", [(395, 1378, 1260), (2000, 700, 700), (256, 3000, 2100)])
def test_loss_of_confident_logits(size, confidence, bit):
    """inputs that are mostly 0, so that a channel's gradient at its own label meets none of some: those are made of the far smaller ones.  The weights are multiples of 1/64, so the logits are exact,
    and a probability is off by 48 roundings: exp, the sum of up to 3000 in tiles, the quotient (32), and what follows"""
    from binarybrain_amd import ops
    inputs, channels, frames = size
    rng = np.random.default_rng(5)
    label = rng.integers(0, channels, (1, frames)).astype(np.int32)
    on = rng.random((inputs, frames)) < 0.05
    W = (np.round(rng.standard_normal((channels, inputs)) * 64 * 8.0 / np.sqrt(0.05 * inputs)) / 64).astype(F32)
    b = np.zeros(channels, F32)
    for k in range(min(inputs, 64)):                # an input of its own for the labels of a kind, which makes them more certain
        on[k] = label[0] % 64 == k
        W[:, k] = 0.0
        W[k::64, k] = confidence
    values = on.astype(np.float64)
    pitch = (frames + 31) // 32 * 32
    if bit:
        x = np.packbits(np.pad(on.astype(np.uint8), ((0, 0), (0, pitch - frames))), axis=1, bitorder="little").view(np.int32)
        loss, dx, dW, db = ops.bit_loss_dense_softmax_cross_entropy(dev(x), dev(W), dev(b), dev(label), frames, pitch)
    else:
        loss, dx, dW, db = ops.loss_dense_softmax_cross_entropy(dev(on.astype(F32)), dev(W), dev(b), dev(label), frames)
    W64 = W.astype(np.float64)
    want, dz, want_dx, want_dW, want_db = exact_loss(values, W64, b.astype(np.float64), label[0], np.ones(frames), float(frames))
    dz_off = cases.loss_bounds(values, W64, b, dz, np.ones(frames), float(frames), np.zeros((channels, frames)))
    # (what is added there for every channel is the rounding of p - 1 at the label alone)
    dz_off -= np.where(np.arange(channels)[:, None] == label, 0.0, 8 * U / frames)
    near(host(dW), want_dW, even_bound(dz, values.T) + dz_off @ values.T + 2.0 ** -140, "dW")
    near(host(dx)[:, :frames], want_dx, even_bound(W64.T, dz) + np.abs(W64.T) @ dz_off + 2.0 ** -140, "dx")
