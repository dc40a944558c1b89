"""GPU: elements of large dense products that are formed again, straight from the operands.  An infinity or a NaN in an operand: the elements that it reaches are what the formula says, in every
form of a product, all others have the bits that they have without it, and a call that holds some costs no multiple of a plain one."""
import numpy as np
import pytest

import test_gpu_dense as cases
from dense_reference import U, bits_of, loss as exact_loss, product_bound
from test_gpu_dense import dev, host, near, rows

pytestmark = pytest.mark.gpu

F32 = np.float32
# (inputs, outputs, frames): tiles of each size, whole and with a shared k axis, odd ends
SIZES = [(300, 2600, 2500), (640, 530, 1100), (1103, 640, 1300), (145, 21806, 548)]


def differ_only_at(a, b, where):
    """bits, NaN among them"""
    same = a.view(np.int32) == b.view(np.int32)
    return bool(np.all(same[~where]))


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_forward_leaves_the_others_alone(size, bit):
    """NaN and infinities in two outputs' weights and in two frames"""
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    rng, x, values, W, b = cases.layer(3, inputs, outputs, frames, bit, (frames + 31) // 32 * 32)
    r = rows(rng, outputs, frames, frames)

    def call(x, W):
        if bit:
            return host(ops.bit_dense_affine_forward(dev(x), dev(W), dev(b), frames, frames, residual=dev(r)))
        return host(ops.dense_affine_forward(dev(x), dev(W), dev(b), frames, residual=dev(r)))[:, :frames]
    plain = call(x, W)
    V, z = W.copy(), x.copy()
    V[outputs // 2, 7], V[outputs - 1, 3] = np.nan, np.inf
    reached = np.zeros((outputs, frames), bool)
    reached[[outputs // 2, outputs - 1]] = True
    if not bit:
        z[5, frames // 3], z[9, frames - 1] = np.inf, np.nan
        reached[:, [frames // 3, frames - 1]] = True
    odd = call(z, V)
    assert differ_only_at(plain, odd, reached)
    with np.errstate(all="ignore"):
        want = V.astype(np.float64) @ (bits_of(z, frames) if bit else z[:, :frames].astype(np.float64)) + b.astype(np.float64)[:, None] + r[:, :frames]
    assert np.array_equal(np.isnan(odd), np.isnan(want)) and np.array_equal(np.isinf(odd), np.isinf(want)) and np.array_equal(np.signbit(odd[np.isinf(odd)]), np.signbit(want[np.isinf(want)]))
    # (a bit of 0 times an infinity is none either, a bit times NaN: every element reached is not finite)
    assert not np.any(np.isfinite(odd[reached]))


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_forward_to_bits_leaves_the_others_alone(size, bit):
    """sums of multiples of 1/64 are exact, so each bit is known; one of a NaN is 0, one of plus infinity 1"""
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    rng = np.random.default_rng(5)
    pitch = (frames + 31) // 32 * 32
    words = rng.integers(-2 ** 31, 2 ** 31, (inputs, pitch // 32)).astype(np.int32)
    values = bits_of(words, frames) if bit else rng.integers(-8, 9, (inputs, frames)) / 4.0 + 0.125
    W = (rng.integers(-16, 17, (outputs, inputs)) / 16.0).astype(F32)
    W[3, 4], W[outputs - 2, 1] = np.nan, np.inf
    x = np.zeros((inputs, pitch), F32)
    x[:, :frames] = values
    with np.errstate(all="ignore"):
        z = W.astype(np.float64) @ values
    got = host(ops.bit_dense_affine_forward_bits(dev(words), dev(W), None, frames) if bit else ops.dense_affine_forward_bits(dev(x), dev(W), None, frames))
    assert np.array_equal(bits_of(got, frames), np.where(np.isnan(z), 0, z > 0))


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", [(300, 2600, 1100), (700, 600, 1200), (1024, 1001, 1000), (2048, 4300, 1500)])
def test_backward_leaves_the_others_alone(size, bit):
    """NaN in one gradient: its output's row of dW, db and its frame's column of dx; gradients are added to what is there"""
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    rng, x, values, W, b = cases.layer(4, inputs, outputs, frames, bit, (frames + 31) // 32 * 32)
    dy = rows(rng, outputs, frames, frames)
    y = np.maximum(rows(rng, outputs, frames, frames), 0.0)
    y[11, 20], y[outputs - 1, frames - 1] = 1.0, 1.0
    there = rng.standard_normal(W.shape).astype(F32), rng.standard_normal(outputs).astype(F32)
    call = ops.bit_dense_affine_backward if bit else ops.dense_affine_backward

    def gradients(dy):
        out = call(dev(x), dev(dy), dev(W), frames, activation="relu", y=dev(y), dW=dev(there[0]), db=dev(there[1]), want_dr=True)
        return [host(t)[:, :frames] if k in (0, 3) else host(t) for k, t in enumerate(out)]
    plain = gradients(dy)
    odd_dy = dy.copy()
    odd_dy[11, 20], odd_dy[outputs - 1, frames - 1] = np.nan, np.inf
    odd = gradients(odd_dy)
    at = [np.zeros(t.shape, bool) for t in plain]
    at[0][:, [20, frames - 1]] = at[1][[11, outputs - 1]] = True
    at[2][[11, outputs - 1]] = at[3][11, 20] = at[3][outputs - 1, frames - 1] = True
    for k in range(4):
        assert differ_only_at(plain[k], odd[k], at[k]), k
    assert np.isnan(odd[0][:, 20]).all() and np.isnan(odd[1][11]).all() and not np.isfinite(odd[0][:, frames - 1]).any()
    if not bit:
        assert np.array_equal(odd[1][outputs - 1], np.copysign(np.inf, x[:, frames - 1]).astype(F32))


# (inputs, channels, frames): straight, packed whole and with a shared k axis for the logits
LOSS_SIZES = [(40, 50, 60), (395, 1378, 1260), (2000, 700, 700), (64, 2500, 2000)]


@pytest.mark.parametrize("size", LOSS_SIZES)
def test_a_weight_of_minus_infinity_closes_a_channel(size):
    """where its input is positive: the same loss, dW, db in every form; dx of that input is no number, as 0 times infinity is"""
    from binarybrain_amd import ops
    inputs, channels, frames = size
    rng, x, values, W, b = cases.layer(7, inputs, channels, frames, False, frames)
    x[2] = np.abs(x[2]) + 0.1
    values = x[:, :frames].astype(np.float64)
    closed = np.zeros(channels, bool)
    closed[[9, 40]] = True
    W[9, 2] = W[40, 2] = -np.inf
    label = rng.integers(0, 9, (1, frames)).astype(np.int32)
    loss, dx, dW, db = ops.loss_dense_softmax_cross_entropy(dev(x), dev(W), dev(b), dev(label), frames)
    keep = ~closed
    want, dz, want_dx, want_dW, want_db = exact_loss(values, W[keep].astype(np.float64), b[keep].astype(np.float64), label[0], np.ones(frames), float(frames))
    others = np.arange(inputs) != 2
    for got, exact in ((host(loss)[0], want), (host(dW)[keep], want_dW), (host(db)[keep], want_db)):
        assert np.linalg.norm(got - exact) <= 1e-6 * np.linalg.norm(exact)
    assert not host(dW)[closed].any() and not host(db)[closed].any()
    assert np.isnan(host(dx)[2]).all()
    whole = W.copy()
    whole[closed] = 0.0
    exact = whole.astype(np.float64)[keep].T @ dz
    exact += W[closed][:, others].astype(np.float64).sum() * 0
    assert np.linalg.norm(host(dx)[others] - exact[others]) <= 1e-6 * np.linalg.norm(exact[others])


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", [(1024, 4096, 4096), (640, 530, 1100)])
def test_operands_full_of_nan_cost_no_multiple(size, bit):
    """a product on the fp32 matrix instructions behind one of halves, plus what one wavefront of the longest chain takes: at most ten times a plain call (a chain per element was hundreds)"""
    import torch
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    rng, x, values, W, b = cases.layer(8, inputs, outputs, frames, bit, (frames + 31) // 32 * 32)
    x, V = dev(x), W.copy()
    V[::3, inputs - 1] = np.nan                 # behind the last k, where no early end helps
    call = (lambda W: ops.bit_dense_affine_forward(x, W, None, frames, frames)) if bit else (lambda W: ops.dense_affine_forward(x, W, None, frames))

    def seconds(W):
        W = dev(W)
        call(W)
        torch.cuda.synchronize()
        a, z = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(3):
            y = call(W)
        z.record()
        torch.cuda.synchronize()
        return a.elapsed_time(z), host(y)[:, :frames]
    plain, odd = seconds(W), seconds(V)
    assert np.isnan(odd[1][::3]).all() and np.array_equal(odd[1][1::3], plain[1][1::3])
    assert odd[0] <= 10 * plain[0] + 3, (plain[0], odd[0])


@pytest.mark.parametrize("size", [(1024, 4096, 4096), (1500, 1024, 1024)])
def test_operands_that_are_all_nan_are_done_at_once(size):
    """whole tiles, and a shared k axis: at most twice a plain call and what the launches behind it take"""
    import torch
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    x, W = torch.randn((inputs, frames), device="cuda"), torch.randn((outputs, inputs), device="cuda")

    def milliseconds(W):
        best = 1e9
        for _ in range(3):
            a, z = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            y = ops.dense_affine_forward(x, W, None, frames)
            z.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(z))
        return best, y
    plain, odd = milliseconds(W)[0], milliseconds(torch.full_like(W, float("nan")))
    assert bool(odd[1].isnan().all()) and odd[0] <= 2 * plain + 0.3, (plain, odd[0])
