"""GPU parity of the operators at the head of a network — LayerNormalization, TopLogits, LossDistillation, CategoricalSampling — through the
Python calls, against their definitions in 64 bits (head_reference.py).

Whole numbers (channels, drawn categories) have to be equal.  Floating results are held to what their roundings allow, U = 2^-24 each:
  mean      a chain of at most 100 roundings of values no larger than max|x|;
  rstd      squares, a chain of at most 100 additions of positive terms, root and quotient: 128 U relative;
  y         the above through (x - mean) rstd gamma + beta, and four roundings of its own;
  dx        sums over nodes of terms |g| and |g xh| in chains of at most 200: 200 U times their mean, times rstd; eight roundings of its own terms;
  dgamma    a chain of at most 200 over |dy xh|, whose terms carry three roundings; dbeta likewise;
  p, q      the exponent (y - max) log2(e) / T carries two roundings, so exp is off by 2 U |y - max| / T and its own 4 U; sums of at most 300 terms in a chain;
  loss      the sum of q (log q - log p): terms of size |z| + |y| over T + log(channels), 400 U of them."""
import numpy as np
import pytest

import head_reference as ref
from head_reference import U
from util import dev, host

pytestmark = pytest.mark.gpu
F32 = np.float32


@pytest.fixture(scope="module")
def ops():
    from binarybrain_amd import ops as o
    return o


def padded(a, stride, fill=np.nan):
    """rows of `stride`, what lies behind the frames filled with a value that would show"""
    out = np.full((a.shape[0], stride), fill, a.dtype)
    out[:, :a.shape[1]] = a
    return out


def pack(bits, words):
    """[nodes, frames] of 0 / 1 -> [nodes, words] int32, all bits behind the last frame set"""
    n, f = bits.shape
    full = np.ones((n, words * 32), np.uint8)
    full[:, :f] = bits
    return np.packbits(full, axis=1, bitorder="little").view(np.int32).copy()


def near(got, want, tol, what):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    off = np.abs(got - want)
    assert np.all(off <= tol), "%s: %.3g off, %.3g allowed" % (what, np.max(off - tol), np.max(tol))


# ---- layer normalisation -----------------------------------------------------------------------------------------------------------
NORM_SHAPES = [
    # nodes, frames, stride
    (1, 1, 1), (2, 1, 64), (1, 5, 8), (3, 3, 3), (7, 64, 64), (64, 63, 64), (65, 65, 65), (100, 130, 132), (129, 257, 260),
    (1000, 1, 1), (1024, 1, 64), (4096, 2, 4), (16384, 1, 64), (5, 5001, 5004), (2, 20000, 20000), (777, 101, 103), (1531, 259, 320),
    (6000, 33, 36), (333, 4098, 4224),
]


@pytest.mark.parametrize("shape", NORM_SHAPES)
@pytest.mark.parametrize("bit", [False, True])
def test_layer_norm(ops, shape, bit):
    nodes, F, stride = shape
    rng = np.random.default_rng(nodes * 7 + F)
    gamma, beta = (1 + 0.3 * rng.standard_normal(nodes)).astype(F32), rng.standard_normal(nodes).astype(F32)
    if bit:
        x = (rng.random((nodes, F)) < 0.3).astype(np.uint8)
        y, mean, rstd = ops.bit_layer_normalization_forward(dev(pack(x, (stride + 31) // 32 + 1)), dev(gamma), dev(beta), F, stride)
    else:
        x = (rng.standard_normal((nodes, F)) * rng.uniform(0.5, 3, F) + rng.uniform(-4, 4, F)).astype(F32)
        y, mean, rstd = ops.layer_normalization_forward(dev(padded(x, stride)), dev(gamma), dev(beta), F)
    wy, wmean, wrstd = ref.layer_norm(x, gamma, beta, float(F32(1e-5)))
    check_norm(x, gamma, beta, host(y)[:, :F], host(mean), host(rstd), wy, wmean, wrstd)


def check_norm(x, gamma, beta, y, mean, rstd, wy, wmean, wrstd):
    x = x.astype(np.float64)
    tol_mean = 100 * U * np.abs(x).max(0)
    near(mean, wmean, tol_mean, "mean")
    # (x - mean)^2 is taken about a mean that is off by tol_mean: the variance moves by its square
    near(rstd, wrstd, 128 * U * wrstd + 0.5 * wrstd ** 3 * tol_mean ** 2 + 1e-30, "rstd")
    g = np.abs(gamma.astype(np.float64))[:, None]
    hat = np.abs(x - wmean) * wrstd
    near(y, wy, g * (wrstd * tol_mean + hat * (132 * U + 0.5 * wrstd ** 2 * tol_mean ** 2)) + 4 * U * (np.abs(wy) + np.abs(beta.astype(np.float64))[:, None]), "y")


def test_layer_norm_without_weights_or_statistics(ops):
    rng = np.random.default_rng(3)
    x = rng.standard_normal((50, 70)).astype(F32)
    y, mean, rstd = ops.layer_normalization_forward(dev(x), None, None, 70, want_statistics=False)
    assert mean is None and rstd is None
    one, zero = np.ones(50, F32), np.zeros(50, F32)
    near(host(y), ref.layer_norm(x, one, zero, 1e-5)[0], 2e-5, "y")          # 132 U times hat <= 5, and the mean's 100 U times 5
    y, _, _ = ops.layer_normalization_forward(dev(x), dev(one), None, 70)
    near(host(y), ref.layer_norm(x, one, zero, 1e-5)[0], 2e-5, "y")


@pytest.mark.parametrize("offset", [0.0, 1e3, 1e5])
def test_layer_norm_of_a_large_mean(ops, offset):
    """values far from zero: a sum of squares would lose the variance altogether at 1e5"""
    rng = np.random.default_rng(4)
    nodes, F = 3000, 70
    x = (offset + rng.standard_normal((nodes, F))).astype(F32)
    one, zero = np.ones(nodes, F32), np.zeros(nodes, F32)
    y, mean, rstd = ops.layer_normalization_forward(dev(padded(x, 72)), dev(one), dev(zero), F)
    check_norm(x, one, zero, host(y)[:, :F], host(mean), host(rstd), *ref.layer_norm(x, one, zero, float(F32(1e-5))))


def test_layer_norm_of_equal_values(ops):
    """no deviation at all: rstd is 1 / sqrt(eps), y is beta"""
    x = np.full((200, 9), 3.25, F32)
    beta = np.arange(200, dtype=F32)
    y, mean, rstd = ops.layer_normalization_forward(dev(x), None, dev(beta), 9, eps=0.25)
    assert np.array_equal(host(y), np.repeat(beta[:, None], 9, 1)) and np.all(host(mean) == 3.25) and np.all(host(rstd) == 2.0)


def test_layer_norm_keeps_a_frame_to_itself(ops):
    """infinities and what is not a number stay in their frame"""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((300, 40)).astype(F32)
    clean = host(ops.layer_normalization_forward(dev(x), None, None, 40)[0])
    bad = x.copy()
    bad[17, 3], bad[250, 21], bad[0, 22] = np.nan, np.inf, -np.inf
    y = host(ops.layer_normalization_forward(dev(bad), None, None, 40)[0])
    touched = np.isin(np.arange(40), (3, 21, 22))
    assert np.array_equal(y[:, ~touched], clean[:, ~touched]) and np.all(np.isnan(y[:, touched]).any(0))


@pytest.mark.parametrize("shape", NORM_SHAPES)
@pytest.mark.parametrize("bit", [False, True])
def test_layer_norm_backward(ops, shape, bit):
    nodes, F, stride = shape
    rng = np.random.default_rng(nodes * 11 + F)
    gamma = (1 + 0.3 * rng.standard_normal(nodes)).astype(F32)
    dy = rng.standard_normal((nodes, F)).astype(F32)
    if bit:
        x = (rng.random((nodes, F)) < 0.5).astype(np.uint8)
        given = dev(pack(x, (stride + 31) // 32))
    else:
        x = (rng.standard_normal((nodes, F)) + rng.uniform(-2, 2, F)).astype(F32)
        given = dev(padded(x, stride + 4))
    _, mean, rstd = ref.layer_norm(x, gamma, gamma, 1e-5)
    mean, rstd = mean.astype(F32), rstd.astype(F32)
    call = ops.bit_layer_normalization_backward if bit else ops.layer_normalization_backward
    dx, dgamma, dbeta = call(given, dev(padded(dy, stride)), dev(gamma), dev(mean), dev(rstd), F)
    wdx, wdg, wdb = ref.layer_norm_backward(x, dy, gamma, mean, rstd)
    check_norm_backward(x, dy, gamma, mean, rstd, host(dx)[:, :F], host(dgamma), host(dbeta), wdx, wdg, wdb)
    # given gradients are added to
    dg, db = dev(np.full(nodes, 2.0, F32)), dev(np.full(nodes, -3.0, F32))
    again = call(given, dev(padded(dy, stride)), dev(gamma), dev(mean), dev(rstd), F, dgamma=dg, dbeta=db)
    assert np.array_equal(host(again[0])[:, :F], host(dx)[:, :F])
    assert np.array_equal(host(dg), F32(2) + host(dgamma)) and np.array_equal(host(db), F32(-3) + host(dbeta))
    # and may be left out
    alone = call(given, dev(padded(dy, stride)), dev(gamma), dev(mean), dev(rstd), F, want_weights=False)
    assert alone[1] is None and alone[2] is None and np.array_equal(host(alone[0])[:, :F], host(dx)[:, :F])


def check_norm_backward(x, dy, gamma, mean, rstd, dx, dgamma, dbeta, wdx, wdg, wdb):
    x, dy, mean, rstd = (a.astype(np.float64) for a in (x, dy, mean, rstd))
    xh, g = (x - mean) * rstd, dy * gamma.astype(np.float64)[:, None]
    a, b = np.abs(g).mean(0), np.abs(g * xh).mean(0)
    near(dx, wdx, rstd * (8 * U * (np.abs(g) + a + np.abs(xh) * b) + 204 * U * (a + np.abs(xh) * b)), "dx")
    near(dgamma, wdg, 204 * U * np.abs(dy * xh).sum(1), "dgamma")
    near(dbeta, wdb, 200 * U * np.abs(dy).sum(1), "dbeta")


def test_layer_norm_backward_against_differences(ops):
    """the gradient against central differences of the 64-bit forward pass: their error is of second order in the step (1e-4)^2 and U / step of the loss"""
    rng = np.random.default_rng(8)
    x, t = rng.standard_normal((40, 6)), rng.standard_normal((40, 6))
    gamma, beta = 1 + 0.2 * rng.standard_normal(40), rng.standard_normal(40)
    x, t, gamma, beta = (a.astype(F32) for a in (x, t, gamma, beta))
    value = lambda x_, g_, b_: float((ref.layer_norm(x_, np.float64(g_), np.float64(b_), 1e-5)[0] * t).sum())
    _, mean, rstd = ops.layer_normalization_forward(dev(x), dev(gamma), dev(beta), 6)
    dx, dgamma, dbeta = ops.layer_normalization_backward(dev(x), dev(t), dev(gamma), mean, rstd, 6)
    h = 1e-4
    for at in [(0, 0), (17, 3), (39, 5)]:
        e = np.zeros((40, 6)); e[at] = h
        assert abs((value(x + e, gamma, beta) - value(x - e, gamma, beta)) / (2 * h) - float(host(dx)[at])) < 1e-4
        e = np.zeros(40); e[at[0]] = h
        assert abs((value(x, gamma + e, beta) - value(x, gamma - e, beta)) / (2 * h) - float(host(dgamma)[at[0]])) < 1e-4
        assert abs((value(x, gamma, beta + e) - value(x, gamma, beta - e)) / (2 * h) - float(host(dbeta)[at[0]])) < 1e-4


# ---- the largest logits ------------------------------------------------------------------------------------------------------------
TOP_SHAPES = [
    # channels, pixels, frames, stride, k
    (1, 1, 1, 1, 1), (2, 1, 1, 64, 2), (10, 1, 64, 64, 4), (10, 1, 63, 64, 10), (21, 12, 9, 12, 5), (32, 3, 7, 7, 32), (33, 5, 6, 8, 33), (70, 2, 130, 132, 7),
    (255, 1, 20, 20, 255), (256, 1, 5, 8, 256), (257, 1, 33, 36, 256), (512, 1, 17, 20, 3), (513, 2, 4, 4, 40), (1000, 1, 101, 103, 64), (1001, 1, 18, 64, 17),
    (5000, 1, 3, 4, 256), (20000, 1, 1, 64, 50), (32768, 1, 2, 2, 1), (9000, 1, 260, 260, 20), (4000, 3, 5, 5, 100),
]


def columns(a, rows, pix, frames):
    """[rows * pix, stride] -> [rows, pix * frames]"""
    return a.reshape(rows, pix, -1)[:, :, :frames].reshape(rows, pix * frames)


def as_rows(a, pix, frames, stride, fill):
    """[rows, pix * frames] -> [rows * pix, stride]"""
    return padded(np.ascontiguousarray(a).reshape(-1, frames), stride, fill)


def logits_of(kind, rng, shape):
    if kind == "random":
        return (3 * rng.standard_normal(shape)).astype(F32)
    if kind == "equal":                                                      # a handful of values: nearly all are ties
        return rng.integers(-2, 3, shape).astype(F32)
    if kind == "constant":
        return np.full(shape, -1.5, F32)
    if kind == "ascending":                                                  # every channel is above all before it
        return (np.arange(shape[0])[:, None] + rng.random(shape) * 0.5).astype(F32)
    if kind == "descending":
        return (-np.arange(shape[0])[:, None] + rng.random(shape) * 0.5).astype(F32)
    y = (3 * rng.standard_normal(shape)).astype(F32)                         # "special"
    some = rng.random(shape)
    y[some < 0.3] = -np.inf
    y[(some > 0.3) & (some < 0.32)] = np.inf
    y[(some > 0.4) & (some < 0.43)] = np.nan
    y[(some > 0.5) & (some < 0.55)] = -0.0
    y[(some > 0.6) & (some < 0.65)] = 0.0
    y[(some > 0.7) & (some < 0.72)] = np.finfo(F32).min
    y[(some > 0.8) & (some < 0.82)] = 1e-42                                  # (denormal)
    y[:, 0] = -np.inf
    y[:, -1] = np.nan
    return y


def same_values(got, want):
    """equal as numbers (-0 is 0), not-a-number where it is wanted"""
    return np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~np.isnan(want)], want[~np.isnan(want)])


@pytest.mark.parametrize("shape", TOP_SHAPES)
@pytest.mark.parametrize("kind", ["random", "equal", "constant", "ascending", "descending", "special"])
def test_top_logits(ops, shape, kind):
    C, P, F, stride, k = shape
    y = logits_of(kind, np.random.default_rng(C + F), (C, P * F))
    index, logit = ops.top_logits(dev(as_rows(y, P, F, stride, np.inf)), k, C, P, F)
    wi, wv = ref.top_logits(y, k)
    gi, gv = columns(host(index), k, P, F), columns(host(logit), k, P, F)
    assert np.array_equal(gi, wi) and same_values(gv, wv)


# ---- distillation ------------------------------------------------------------------------------------------------------------------
DISTILL_SHAPES = [
    # channels, pixels, frames, stride, k
    (1, 1, 1, 1, 1), (2, 1, 1, 64, 1), (10, 1, 64, 64, 4), (10, 1, 63, 64, 10), (21, 12, 9, 12, 5), (33, 5, 6, 8, 33), (70, 2, 130, 132, 7), (255, 1, 20, 20, 200),
    (513, 2, 4, 4, 40), (1001, 1, 101, 103, 17), (5000, 1, 3, 4, 256), (20000, 1, 1, 64, 50), (3000, 1, 260, 260, 20), (2000, 3, 5, 5, 100),
]


def distill_case(rng, C, n, k, scale=3.0):
    y = (scale * rng.standard_normal((C, n))).astype(F32)
    teacher = (y + rng.standard_normal((C, n))).astype(F32)
    index, z = ref.top_logits(teacher, k)
    w = (rng.random(n) + 0.5).astype(F32)
    return y, index.copy(), z.astype(F32), w


def check_distill(y, index, z, w, t, weight_sum, dy, loss):
    wdy, wloss = ref.distillation(y, index, z, w, t, weight_sum)
    y64, z64 = y.astype(np.float64), z.astype(np.float64)
    C = y.shape[0]
    far = lambda a: np.abs(a - np.max(np.where(np.isfinite(a), a, -np.inf), 0)) / t
    e = np.exp(-far(y64))
    p = e / e.sum(0)
    coefficient = np.abs(w.astype(np.float64)) * t / abs(weight_sum)
    d = np.where(np.isfinite(far(y64)), far(y64), 0.0)
    # q <= 1; a listed channel carries the roundings of both shares
    listed = np.zeros(y.shape, bool)
    for f in range(y.shape[1]):
        at = index[:, f]
        listed[at[(at >= 0) & (at < C)], f] = True
    zspan = np.max(np.where(np.isfinite(z64), np.abs(z64 - np.max(np.where(np.isfinite(z64), z64, -np.inf), 0)), 0.0), 0) / t
    tol = coefficient * (p * (2 * d + 310) + np.where(listed, np.minimum(1.0, np.abs(wdy) / np.maximum(coefficient, 1e-300) + p) * (2 * zspan + 310), 0.0)) * U
    near(dy, wdy, tol + 1e-38, "dy")
    size = 1 + np.log(C) + np.abs(np.where(np.isfinite(y64), y64, 0)).max(0) / t + 2 * np.abs(np.where(np.isfinite(z64), z64, 0)).max(0) / t
    near(loss, wloss, np.abs(w) * t * t * 400 * U * size, "loss")


@pytest.mark.parametrize("shape", DISTILL_SHAPES)
@pytest.mark.parametrize("t", [1.0, 0.25, 4.0])
def test_distillation(ops, shape, t):
    C, P, F, stride, k = shape
    rng = np.random.default_rng(C * 3 + F)
    y, index, z, w = distill_case(rng, C, P * F, k)
    index[k // 2 + 1:, ::3] = -1                                            # shorter lists
    w[5::7] = 0.0
    ws = float(max(w.astype(np.float64).sum(), 1.0))
    dy, loss = ops.loss_distillation(dev(as_rows(y, P, F, stride, np.nan)), dev(as_rows(index, P, F, stride + 4, 0)), dev(as_rows(z, P, F, stride + 4, np.nan)), C, P, F,
                                     temperature=t, weight=dev(as_rows(w[None], P, F, stride, np.nan)), weight_sum=ws)
    check_distill(y, index, z, w, t, float(F32(ws)), columns(host(dy), C, P, F), columns(host(loss), 1, P, F)[0])


def test_distillation_defaults(ops):
    """weight None: 1 everywhere, and the sum of the weights is the number of places"""
    rng = np.random.default_rng(12)
    y, index, z, _ = distill_case(rng, 50, 2 * 30, 8)
    dy, loss = ops.loss_distillation(dev(as_rows(y, 2, 30, 32, 0)), dev(as_rows(index, 2, 30, 32, 0)), dev(as_rows(z, 2, 30, 32, 0)), 50, 2, 30)
    check_distill(y, index, z, np.ones(60, F32), 1.0, 60.0, columns(host(dy), 50, 2, 30), columns(host(loss), 1, 2, 30)[0])
    w = (rng.random((2, 32)) + 0.1).astype(F32)
    dy, loss = ops.loss_distillation(dev(as_rows(y, 2, 30, 32, 0)), dev(as_rows(index, 2, 30, 32, 0)), dev(as_rows(z, 2, 30, 32, 0)), 50, 2, 30, weight=dev(w))
    w = w[:, :30].reshape(-1)
    check_distill(y, index, z, w, 1.0, float(w.astype(np.float64).sum()), columns(host(dy), 50, 2, 30), columns(host(loss), 1, 2, 30)[0])


@pytest.mark.parametrize("C", [30, 700])
def test_distillation_of_odd_lists(ops, C):
    """no entries, entries of minus infinity, channels that are none, channels named twice and three times, whole lists of one channel"""
    rng = np.random.default_rng(13)
    y, index, z, w = distill_case(rng, C, 40, 12)
    index[:, 0] = -1                                                         # nothing at all
    z[:, 1] = -np.inf                                                        # nothing but minus infinity
    index[3:6, 2] = C; index[7, 2] = 1 << 30; index[8, 2] = -(1 << 31)       # no channels of this layer
    index[5, 3] = index[2, 3]                                                # twice
    index[6, 4] = index[11, 4] = index[0, 4]                                 # three times
    index[:, 5] = 7                                                          # one channel, twelve times
    z[4:, 6] = -np.inf                                                       # part of a list
    index[1:, 7] = -1                                                        # a list of one
    index[:-1, 8] = -1                                                       # its last entry
    z[:, 9] = 1e30                                                           # equal, and large
    z[0, 10] = np.inf                                                        # all of the share
    y[:, 11] = 1e30
    y[:, 12] = -np.inf; y[index[0, 12], 12] = 0.5; index[1:, 12] = -1        # a mask that leaves one channel, the listed one
    dy, loss = ops.loss_distillation(dev(y), dev(index), dev(z), C, 1, 40, temperature=2.0, weight=dev(w[None]), weight_sum=10.0)
    dy, loss = host(dy), host(loss)[0]
    assert not dy[:, :2].any() and not loss[:2].any()
    check_distill(y, index, z, w, 2.0, 10.0, dy, loss)


def test_distillation_of_masked_logits(ops):
    """-inf in masked channels: no gradient there; a listed one is an infinite loss, its gradient finite; a weight of 0 leaves nothing of anything"""
    rng = np.random.default_rng(14)
    y, index, z, w = distill_case(rng, 600, 20, 5)
    y[rng.random(y.shape) < 0.5] = -np.inf
    y[index, np.arange(20)] = 1.0
    y[index[2, 3], 3] = -np.inf
    y[:, 4] = np.nan; w[4] = 0
    y[:, 5] = -np.inf; w[5] = 0
    z[:, 6] = np.nan; w[6] = 0
    dy, loss = ops.loss_distillation(dev(y), dev(index), dev(z), 600, 1, 20, weight=dev(w[None]), weight_sum=4.0)
    dy, loss = host(dy), host(loss)[0]
    assert np.isposinf(loss[3]) and np.all(np.isfinite(dy)) and not dy[:, 4:7].any() and not loss[4:7].any()
    assert np.all(dy[np.isneginf(y) & (np.arange(600)[:, None] != index[2, 3])] == 0.0)
    keep = np.array([f for f in range(20) if f not in (3, 4, 5, 6)])
    check_distill(y[:, keep], index[:, keep], z[:, keep], w[keep], 1.0, 4.0, dy[:, keep], loss[keep])


def test_distillation_keeps_a_frame_to_itself(ops):
    rng = np.random.default_rng(15)
    y, index, z, w = distill_case(rng, 90, 24, 6)
    call = lambda: [host(a) for a in ops.loss_distillation(dev(y), dev(index), dev(z), 90, 1, 24, weight=dev(w[None]), weight_sum=4.0)]
    clean = call()
    y[3, 2], y[4, 9], z[2, 17] = np.nan, np.inf, np.nan
    got = call()
    touched = np.isin(np.arange(24), (2, 9, 17))
    assert np.array_equal(got[0][:, ~touched], clean[0][:, ~touched]) and np.array_equal(got[1][:, ~touched], clean[1][:, ~touched])
    assert np.all(np.isnan(got[1][0, touched]))


def test_distillation_gradient_against_differences(ops):
    rng = np.random.default_rng(16)
    y, index, z, w = distill_case(rng, 40, 5, 6, scale=1.0)
    dy, _ = ops.loss_distillation(dev(y), dev(index), dev(z), 40, 1, 5, temperature=2.0, weight=dev(w[None]), weight_sum=3.0)
    value = lambda y_: ref.distillation(y_, index, z, w, 2.0, 3.0)[1].sum() / 3.0
    h = 1e-4
    for at in [(int(index[0, 0]), 0), (int(index[5, 1]), 1), (0, 2), (39, 4)]:
        e = np.zeros(y.shape); e[at] = h
        assert abs((value(y + e) - value(y.astype(np.float64) - e)) / (2 * h) - float(host(dy)[at])) < 1e-5


# ---- sampling ----------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", TOP_SHAPES)
@pytest.mark.parametrize("rule", [(1.0, 1.0, 0.0), (0.7, 0.9, 0.0), (1.3, 1.0, 0.1), (2.0, 0.6, 0.02)])
def test_sampling(ops, shape, rule):
    C, P, F, stride, k = shape
    t, top_p, min_p = rule
    for kind in ("random", "equal", "special"):
        rng = np.random.default_rng(C + 5 * F)
        y, u = logits_of(kind, rng, (C, P * F)), rng.random(P * F).astype(F32)
        u[0], u[-1] = 0.0, np.nextafter(F32(1), F32(0))
        category, share = ops.categorical_sampling(dev(as_rows(y, P, F, stride, np.inf)), dev(as_rows(u[None], P, F, stride, np.nan)), C, P, F, temperature=t, top_size=k,
                                                   top_p=top_p, min_p=min_p)
        wc, ws = ref.sampling(y, u, t, k, top_p, min_p)
        gc, gs = columns(host(category), 1, P, F)[0], columns(host(share), 1, P, F)[0]
        assert np.array_equal(gc, wc), kind
        near(gs, ws, 2 * U * ws, kind)                                       # one rounding to 32 bits


def test_sampling_of_nothing(ops):
    """a mask that leaves no channel: no category; one that leaves one: that one, whatever is drawn"""
    y = np.full((300, 6), -np.inf, F32)
    y[123, 1] = -7.0
    y[:, 2] = np.nan
    y[5, 3], y[9, 3] = np.inf, np.inf
    y[44, 4] = np.finfo(F32).min
    u = np.full((1, 6), 0.99, F32)
    category, share = ops.categorical_sampling(dev(y), dev(u), 300, 1, 6, top_size=20)
    assert host(category)[0].tolist() == [-1, 123, -1, 9, 44, -1] and host(share)[0].tolist() == [0.0, 1.0, 0.0, 0.5, 1.0, 0.0]


def test_sampling_follows_the_distribution(ops):
    """as many draws of one distribution as frames: counts within five standard deviations"""
    rng = np.random.default_rng(20)
    logits, F = np.log(np.array([0.5, 0.25, 0.15, 0.1], F32)), 40000
    y = np.repeat(logits[:, None], F, 1)
    category, _ = ops.categorical_sampling(dev(y), dev(rng.random((1, F)).astype(F32)), 4, 1, F, top_size=4, want_share=False)
    p = np.array([0.5, 0.25, 0.15, 0.1])
    assert np.all(np.abs(np.bincount(host(category)[0], minlength=4) - F * p) < 5 * np.sqrt(F * p * (1 - p)))


def test_one_logit_is_the_largest(ops):
    rng = np.random.default_rng(21)
    y = logits_of("equal", rng, (90, 33))
    category, share = ops.categorical_sampling(dev(y), dev(rng.random((1, 33)).astype(F32)), 90, 1, 33, top_size=1)
    assert np.array_equal(host(category)[0], y.argmax(0)) and np.all(host(share) == 1.0)


# ---- edges -------------------------------------------------------------------------------------------------------------------------
def test_buffers_beyond_4_gib(ops):
    """offsets that do not fit 32 bits: 70000 rows of 16384 frames; the first and last columns against 64 bits, the last rows written"""
    import torch
    nodes, F, k = 70000, 16384, 3
    gen = torch.Generator(device="cuda"); gen.manual_seed(1)
    x = torch.randn((nodes, F), generator=gen, device="cuda")
    some = [0, 1, 4095, 8190, F - 2, F - 1]
    v = host(x[:, some])
    one, zero = np.ones(nodes, F32), np.zeros(nodes, F32)
    y, mean, rstd = ops.layer_normalization_forward(x, dev(one), dev(zero), F)
    check_norm(v, one, zero, host(y[:, some]), host(mean)[some], host(rstd)[some], *ref.layer_norm(v, one, zero, float(F32(1e-5))))
    dx, dgamma, dbeta = ops.layer_normalization_backward(x, y, dev(one), mean, rstd, F)
    wdx, _, _ = ref.layer_norm_backward(v, host(y[:, some]), one, host(mean)[some], host(rstd)[some])
    g, at_mean, at_rstd = (host(a).astype(np.float64) for a in (y[:, some], mean[some], rstd[some]))
    xh = (v - at_mean) * at_rstd
    a, b = np.abs(g).mean(0), np.abs(g * xh).mean(0)
    near(host(dx[:, some]), wdx, at_rstd * (8 * U * (np.abs(g) + a + np.abs(xh) * b) + 204 * U * (a + np.abs(xh) * b)), "dx")
    last = (x[-4:].double() - mean.double()) * rstd.double()
    near(host(dgamma)[-4:], host((y[-4:].double() * last).sum(1)), 204 * U * host((y[-4:].double() * last).abs().sum(1)), "dgamma")
    del y, dx
    index, logit = ops.top_logits(x, k, nodes, 1, F)
    wi, wv = ref.top_logits(v, k)
    assert np.array_equal(host(index[:, some]), wi) and np.array_equal(host(logit[:, some]), wv)
    dy, loss = ops.loss_distillation(x, index, logit, nodes, 1, F, weight_sum=1.0)
    check_distill(v, wi, wv, np.ones(len(some), F32), 1.0, 1.0, host(dy[:, some]), host(loss[:, some])[0])


def test_a_batch_of_padding_only(ops):
    """weights that are all 0, and so is their sum: no loss, no gradient, nothing that is not a number"""
    rng = np.random.default_rng(40)
    for C in (20, 500):
        y, index, z, _ = distill_case(rng, C, 16, 5)
        w = np.zeros((1, 16), F32)
        dy, loss = ops.loss_distillation(dev(y), dev(index), dev(z), C, 1, 16, weight=dev(w))
        assert not host(dy).any() and not host(loss).any()


def test_lists_longer_than_the_channels(ops):
    """a teacher's record may hold more entries than there are channels: most of them name one again"""
    rng = np.random.default_rng(41)
    for C in (4, 60):
        k = 200
        y = rng.standard_normal((C, 24)).astype(F32)
        index, z = rng.integers(-2, C + 2, (k, 24)).astype(np.int32), rng.standard_normal((k, 24)).astype(F32)
        dy, loss = ops.loss_distillation(dev(y), dev(index), dev(z), C, 1, 24, temperature=1.5, weight_sum=2.0)
        check_distill(y, index, z, np.ones(24, F32), 1.5, 2.0, host(dy), host(loss)[0])


def test_numbers_outside_the_unit_interval(ops):
    """u below 0 draws the first of the kept, u of 1 and above the last"""
    y = np.repeat(np.log(np.array([0.1, 0.6, 0.3], F32))[:, None], 4, 1)
    u = np.array([[-1.0, 1.0, 7.0, 0.0]], F32)
    for pad in (0, 50):
        z = np.concatenate([y, np.full((pad, 4), -30.0, F32)])
        category, _ = ops.categorical_sampling(dev(z), dev(u), 3 + pad, 1, 4, top_size=3)
        assert host(category)[0].tolist() == [1, 0, 0, 1]


def test_refusals_on_the_device(ops):
    import torch
    from binarybrain_amd.capi import BbhipError
    x, i, line = torch.zeros(40, 8, device="cuda"), torch.zeros((4, 8), dtype=torch.int32, device="cuda"), torch.zeros(40, device="cuda")
    z, one = torch.zeros(4, 8, device="cuda"), torch.zeros(1, 8, device="cuda")
    for call in (lambda: ops.layer_normalization_forward(x, line[:3], line, 8), lambda: ops.layer_normalization_forward(x, line, line.double(), 8),
                 lambda: ops.layer_normalization_forward(x.double(), line, line, 8), lambda: ops.layer_normalization_forward(x, line, line, 9),
                 lambda: ops.layer_normalization_forward(x, line, line, 0), lambda: ops.layer_normalization_forward(x, line, line, 8, eps=-1.0),
                 lambda: ops.layer_normalization_forward(x.t(), line, line, 8), lambda: ops.bit_layer_normalization_forward(x, line, line, 8, 8),
                 lambda: ops.layer_normalization_backward(x, x[:20], line, line[:8], line[:8], 8), lambda: ops.layer_normalization_backward(x, x, line, line[:7], line[:8], 8),
                 lambda: ops.layer_normalization_backward(x, x, line, line[:8], line[:8], 8, dgamma=line), lambda: ops.top_logits(x, 41, 40, 1, 8),
                 lambda: ops.top_logits(x, 3, 39, 1, 8), lambda: ops.top_logits(x, 0, 40, 1, 8), lambda: ops.loss_distillation(x, i.float(), z, 40, 1, 8),
                 lambda: ops.loss_distillation(x, i, z[:3], 40, 1, 8), lambda: ops.loss_distillation(x, i, z, 40, 1, 8, weight=x), lambda: ops.loss_distillation(x, i, z, 40, 1, 8, temperature=0.0),
                 lambda: ops.loss_distillation(x, i[:3].contiguous(), z[:3].contiguous(), 20, 2, 8), lambda: ops.categorical_sampling(x, one, 40, 1, 8, top_size=0),
                 lambda: ops.categorical_sampling(x, one, 40, 1, 8, top_size=41), lambda: ops.categorical_sampling(x, one, 40, 1, 8, top_size=3, top_p=0.0),
                 lambda: ops.categorical_sampling(x, one, 40, 1, 8, top_size=3, min_p=2.0), lambda: ops.categorical_sampling(x, one, 40, 1, 8, top_size=3, temperature=-1.0),
                 lambda: ops.categorical_sampling(x, torch.zeros(1, 16, device="cuda"), 40, 1, 8, top_size=3)):
        with pytest.raises(BbhipError):
            call()


def test_buffers_that_do_not_start_on_16_bytes(ops):
    """the same bits of whole numbers and selections, results as near as elsewhere, from buffers shifted by one float"""
    import torch
    rng = np.random.default_rng(42)
    shifted = lambda a: torch.cat([torch.zeros(1, dtype=dev(a).dtype, device="cuda"), dev(a).reshape(-1)])[1:].view(a.shape)
    C, F, k = 700, 24, 9
    y, index, z, w = distill_case(rng, C, F, k)
    one, zero = np.ones(C, F32), np.zeros(C, F32)
    t = shifted(y)
    assert t.data_ptr() % 16 == 4 and t.is_contiguous()
    got = ops.layer_normalization_forward(t, shifted(one), shifted(zero), F)
    check_norm(y, one, zero, *(host(a) for a in got), *ref.layer_norm(y, one, zero, float(F32(1e-5))))
    dx, dg, db = ops.layer_normalization_backward(t, shifted(z[:1] + y), shifted(one), got[1], got[2], F)
    check_norm_backward(y, z[:1] + y, one, host(got[1]), host(got[2]), host(dx), host(dg), host(db), *ref.layer_norm_backward(y, z[:1] + y, one, host(got[1]), host(got[2])))
    gi, gv = ops.top_logits(t, k, C, 1, F)
    wi, wv = ref.top_logits(y, k)
    assert np.array_equal(host(gi), wi) and np.array_equal(host(gv), wv)
    dy, loss = ops.loss_distillation(t, shifted(index), shifted(z), C, 1, F, weight=shifted(w[None]), weight_sum=3.0)
    check_distill(y, index, z, w, 1.0, 3.0, host(dy), host(loss)[0])
    u = rng.random((1, F)).astype(F32)
    category, _ = ops.categorical_sampling(t, shifted(u), C, 1, F, top_size=k, top_p=0.8)
    assert np.array_equal(host(category)[0], ref.sampling(y, u[0], 1.0, k, 0.8, 0.0)[0])
