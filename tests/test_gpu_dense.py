"""GPU parity of dense layers and of the loss on top of one against 64 bits, over sizes, pitches, masks and special values."""
import numpy as np
import pytest

from dense_reference import U, activated, bits_of, loss as exact_loss, product_bound, through

pytestmark = pytest.mark.gpu

ACTIVATIONS = ["none", "relu", "sigmoid", "hard_tanh"]


def rows(rng, n, frames, pitch, scale=1.0):
    a = np.full((n, pitch), np.nan, np.float32)         # what lies behind the last frame is nobody's
    a[:, :frames] = rng.standard_normal((n, frames)).astype(np.float32) * scale
    return a


def dev(a, off=False):
    """on the device; `off`: four bytes behind a multiple of 16"""
    import torch
    t = torch.from_numpy(np.ascontiguousarray(a))
    if not off:
        return t.cuda()
    room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
    room[1:].copy_(t.reshape(-1))
    return room[1:].view(t.shape)


def host(t):
    return t.detach().cpu().numpy()


def layer(seed, inputs, outputs, frames, bit, pitch):
    rng = np.random.default_rng(seed)
    if bit:
        words = rng.integers(-2 ** 31, 2 ** 31, (inputs, pitch // 32 + 1)).astype(np.int32)
        x, values = words, bits_of(words, frames)
    else:
        x = rows(rng, inputs, frames, pitch)
        values = x[:, :frames].astype(np.float64)
    W = (rng.standard_normal((outputs, inputs)) / np.sqrt(inputs)).astype(np.float32)
    b = rng.standard_normal(outputs).astype(np.float32)
    return rng, x, values, W, b


# (inputs, outputs, frames, pitch): one of each, edges of tiles and chunks, many inputs, few frames, many frames, sizes that take the other forms of the kernels
SIZES = [(1, 1, 1, 1), (5, 3, 2, 3), (32, 32, 32, 32), (33, 31, 33, 37), (64, 65, 63, 64), (700, 10, 65, 66), (1, 70, 129, 130), (2000, 40, 1, 1), (129, 127, 300, 301),
         (1024, 1001, 250, 256), (257, 513, 1030, 1031), (1500, 300, 2100, 2112), (16, 2050, 515, 516)]


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_forward(size, bit):
    from binarybrain_amd import ops
    inputs, outputs, frames, pitch = size
    for k, activation in enumerate(ACTIVATIONS):
        rng, x, values, W, b = layer(k, inputs, outputs, frames, bit, pitch)
        r = rows(rng, outputs, frames, frames + k) if k % 2 else None
        give = dict(activation=activation, residual=None if r is None else dev(r))
        off = k >= 2
        if bit:
            y = ops.bit_dense_affine_forward(dev(x, off), dev(W, off), dev(b), frames, pitch, **give)
        else:
            y = ops.dense_affine_forward(dev(x, off), dev(W, off), dev(b), frames, **give)
        z = W.astype(np.float64) @ values + b.astype(np.float64)[:, None] + (0 if r is None else r[:, :frames].astype(np.float64))
        # two more roundings (bias, residual) of values up to the sums'; an activation's slope is 1 at most, the sigmoid itself is off by 4 roundings of values up to 1
        bound = product_bound(W.astype(np.float64), values) + 4 * U * (np.abs(z) + np.abs(b)[:, None] + (0 if r is None else np.abs(r[:, :frames]))) + 4 * U
        got = host(y)[:, :frames].astype(np.float64)
        assert y.shape == (outputs, pitch) and np.all(np.abs(got - activated(z, activation)) <= bound), (activation, np.max(np.abs(got - activated(z, activation)) / bound))
        if activation == "none":
            assert np.linalg.norm(got - z) <= 2.0 ** -20 * np.linalg.norm(z)


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", [(5, 3, 2, 32), (129, 127, 300, 320), (300, 70, 1000, 1024), (1024, 520, 1100, 1120)])
def test_forward_to_bits(size, bit):
    """sums of multiples of 1/64 are exact, so the bits are; what lies behind the last frame is 0"""
    from binarybrain_amd import ops
    inputs, outputs, frames, pitch = size
    rng = np.random.default_rng(inputs)
    words = rng.integers(-2 ** 31, 2 ** 31, (inputs, pitch // 32)).astype(np.int32)
    values = bits_of(words, frames) if bit else rng.integers(-8, 9, (inputs, frames)) / 4.0
    W = (rng.integers(-16, 17, (outputs, inputs)) / 16.0).astype(np.float32)
    b = (rng.integers(-16, 17, outputs) / 16.0).astype(np.float32)
    r = np.full((outputs, pitch), np.nan, np.float32)
    r[:, :frames] = rng.integers(-4, 5, (outputs, frames)) / 4.0
    x = np.zeros((inputs, pitch), np.float32)
    x[:, :frames] = values
    call = (lambda **k: ops.bit_dense_affine_forward_bits(dev(words), dev(W), dev(b), frames, **k)) if bit else (lambda **k: ops.dense_affine_forward_bits(dev(x), dev(W), dev(b), frames, **k))
    for residual in (None, r):
        z = W.astype(np.float64) @ values + b[:, None] + (0 if residual is None else residual[:, :frames])
        got = host(call(residual=None if residual is None else dev(residual), y_words=pitch // 32 + 3))
        assert got.shape == (outputs, pitch // 32 + 3) and np.array_equal(bits_of(got, got.shape[1] * 32)[:, :frames], z > 0) and not bits_of(got, got.shape[1] * 32)[:, frames:].any()


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", SIZES)
def test_backward(size, bit):
    from binarybrain_amd import ops
    inputs, outputs, frames, pitch = size
    for k, activation in enumerate(ACTIVATIONS):
        rng, x, values, W, b = layer(50 + k, inputs, outputs, frames, bit, pitch)
        dy = rows(rng, outputs, frames, pitch)
        y = activated(rows(rng, outputs, frames, pitch).astype(np.float64), activation).astype(np.float32)
        dz = through(dy[:, :frames].astype(np.float64), y[:, :frames].astype(np.float64), activation)
        off = k >= 2
        add = k == 1
        dW0, db0 = rng.standard_normal(W.shape).astype(np.float32), rng.standard_normal(outputs).astype(np.float32)
        call = ops.bit_dense_affine_backward if bit else ops.dense_affine_backward
        given = dict(dW=dev(dW0), db=dev(db0)) if add else {}
        dx, dW, db, dr = call(dev(x, off), dev(dy, off), dev(W, off), frames, activation=activation, y=None if activation == "none" else dev(y, off), want_dr=True, **given)
        slack = 4 * U * np.abs(dz)              # (the sigmoid's slope: three roundings)
        W64 = W.astype(np.float64)
        near(host(dx)[:, :frames], W64.T @ dz, product_bound(W64.T, dz) + np.abs(W64.T) @ slack, "dx")
        want = dz @ values.T + (dW0 if add else 0.0)
        near(host(dW), want, product_bound(dz, values.T) + slack @ np.abs(values.T) + 2 * U * np.abs(dW0), "dW")
        near(host(db), dz.sum(1) + (db0 if add else 0.0), product_bound(dz, np.ones((frames, 1)))[:, 0] + slack.sum(1) + 2 * U * np.abs(db0), "db")
        near(host(dr)[:, :frames], dz, slack, "dr")


def near(got, want, bound, what):
    got = got.astype(np.float64)
    assert got.shape == want.shape and np.all(np.abs(got - want) <= bound), (what, float(np.max(np.abs(got - want) / np.maximum(bound, 1e-300))))


def test_backward_of_parts():
    """what is not wanted is not computed, and changes nothing of the rest"""
    from binarybrain_amd import ops
    for inputs, outputs, frames in ((60, 70, 80), (520, 640, 1300)):
        rng, x, values, W, b = layer(3, inputs, outputs, frames, False, frames)
        x, W, dy = dev(x), dev(W), dev(rows(rng, outputs, frames, frames))
        whole = [host(t) for t in ops.dense_affine_backward(x, dy, W, frames, want_dr=True)]
        for keep in range(1, 8):
            part = ops.dense_affine_backward(x, dy, W, frames, want_dx=bool(keep & 1), want_weights=bool(keep & 2), want_dr=bool(keep & 4))
            for t, w, bit in zip(part, whole, (1, 2, 2, 4)):
                assert (t is not None) == bool(keep & bit) and (t is None or np.array_equal(host(t), w))


def test_gradient_is_the_difference_quotient():
    """of sum(c * y), smooth activation: (f(x + h) - f(x - h)) / 2h in 64 bits from the definition"""
    from binarybrain_amd import ops
    rng, x, values, W, b = layer(9, 6, 5, 7, False, 7)
    c = rows(rng, 5, 7, 7)
    y = ops.dense_affine_forward(dev(x), dev(W), dev(b), 7, activation="sigmoid")
    dx, dW, db, dr = ops.dense_affine_backward(dev(x), dev(c), dev(W), 7, activation="sigmoid", y=y, want_dr=True)

    def f(x, W, b, r):
        return (c * activated(W @ x + b[:, None] + r, "sigmoid")).sum()
    at = [values, W.astype(np.float64), b.astype(np.float64), np.zeros((5, 7))]
    for k, got in enumerate((dx, dW, db, dr)):
        got = host(got)
        for i in np.ndindex(got.shape):
            h = np.zeros_like(at[k])
            h[i] = 1e-5
            up, down = [a + h if j == k else a for j, a in enumerate(at)], [a - h if j == k else a for j, a in enumerate(at)]
            assert abs(got[i] - (f(*up) - f(*down)) / 2e-5) <= 1e-5


@pytest.mark.parametrize("size", [(40, 50, 60), (640, 530, 1100)])
def test_special_values(size):
    """infinities and NaN come out where the formula has them, and nowhere else"""
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    rng, x, values, W, b = layer(4, inputs, outputs, frames, False, frames)
    x[3, 5], x[7, 9], x[2, 11], x[4, 11], x[8, 20] = np.inf, -np.inf, np.inf, np.inf, np.nan
    W[6, :], W[9, 3] = 0.0, -np.inf
    x[5, 30] = 3e38
    W[10, 5], W[11, 5] = 1e-30, 8.0
    with np.errstate(all="ignore"):
        want = (W.astype(np.float64) @ x.astype(np.float64) + b[:, None])
        want = np.where(np.abs(want) > 3.5e38, np.copysign(np.inf, want), want)
    got = host(ops.dense_affine_forward(dev(x), dev(W), dev(b), frames))
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isposinf(got), np.isposinf(want)) and np.array_equal(np.isneginf(got), np.isneginf(want))
    fine = np.isfinite(want)
    assert fine.sum() > 0.8 * fine.size
    with np.errstate(all="ignore"):
        finite_x, finite_W = np.where(np.isfinite(x), x, 0).astype(np.float64), np.where(np.isfinite(W), W, 0).astype(np.float64)
    bound = product_bound(finite_W, finite_x) + 4 * U * (np.abs(want) + np.abs(b)[:, None])
    assert np.all(np.abs(got[fine] - want[fine]) <= bound[fine])
    # a closed activation passes 0 whatever dy is
    dy, y = rows(rng, outputs, frames, frames), rows(rng, outputs, frames, frames)
    y = np.maximum(y, 0)
    dy[y == 0] = np.where(rng.random((y == 0).sum()) < 0.5, np.nan, np.inf)
    x = np.where(np.isfinite(x), x, 1).astype(np.float32)
    W = np.where(np.isfinite(W), W, 1).astype(np.float32)
    dz = through(dy.astype(np.float64), y.astype(np.float64), "relu")
    dx, dW, db, dr = ops.dense_affine_backward(dev(x), dev(dy), dev(W), frames, activation="relu", y=dev(y), want_dr=True)
    near(host(dx), W.astype(np.float64).T @ dz, product_bound(W.astype(np.float64).T, dz), "dx")
    near(host(db), dz.sum(1), product_bound(dz, np.ones((frames, 1)))[:, 0], "db")
    near(host(dr), dz, 0 * dz, "dr")


@pytest.mark.parametrize("size", [(48, 40, 50), (512, 512, 1024)])
def test_scales_of_rows(size):
    """rows of any magnitude: each output's error goes by its own row and column"""
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    rng, x, values, W, b = layer(5, inputs, outputs, frames, False, frames)
    W *= (10.0 ** rng.uniform(-15, 15, outputs)).astype(np.float32)[:, None]
    x[:, :frames] *= (10.0 ** rng.uniform(-15, 15, frames)).astype(np.float32)[None]
    W[3], W[4, 1:], x[:, 2] = 0.0, 0.0, 0.0
    got = host(ops.dense_affine_forward(dev(x), dev(W), None, frames)).astype(np.float64)
    want = W.astype(np.float64) @ x.astype(np.float64)
    near(got, want, product_bound(W.astype(np.float64), x.astype(np.float64)) + 1e-44, "y")
    assert not got[3].any() and not got[:, 2].any()


# ---- the loss ------------------------------------------------------------------------------------------------------------------------
def loss_case(seed, inputs, channels, frames, bit, pitch, scale=3.0):
    rng, x, values, W, b = layer(seed, inputs, channels, frames, bit, pitch)
    W *= np.float32(scale)
    label = rng.integers(0, channels, (1, frames + 3)).astype(np.int32)
    weight = (rng.random((1, frames + 1)) + 0.5).astype(np.float32)
    if frames > 2:
        label[0, 1:frames:5] = -1
        label[0, 2:frames:11] = channels
        weight[0, 0:frames:7] = 0.0
    if not bit:
        x[:, :frames][:, (label[0, :frames] < 0)] = np.nan             # frames that do not count hold anything
    w = weight[0, :frames].astype(np.float64)
    counts = (label[0, :frames] >= 0) & (label[0, :frames] < channels)
    values = np.where(counts[None], values, 0.0)
    return x, values, W, b, label, weight, float((w * counts).sum()) or 1.0


def loss_bounds(values, W, b, dz, weight, weight_sum, z_bound):
    """A logit off by e moves a probability by a factor of 1 + 2 e at most (its own and the sum's), the loss by 2 e.  exp, sum, quotient, log: 16 roundings; the sum of C exponents in
    tiles: C more in the worst order."""
    e = z_bound.max(0)
    p = np.abs(dz)
    g = np.abs(weight) / weight_sum
    off = p * (2 * e + (16 + 32) * U)[None] + 8 * U * g[None]           # (at the label p - 1 is rounded)
    # (at the label the probability itself moves, which |dz| = g (1 - p) does not show)
    off += np.where(dz < 0, g[None] * (2 * e + 48 * U)[None], 0.0)
    return off


LOSS_SIZES = [(1, 1, 1, 1), (3, 2, 5, 6), (40, 10, 64, 64), (33, 65, 63, 70), (777, 1001, 300, 300), (20, 5000, 33, 40), (8, 600, 65600, 65600), (64, 2500, 9000, 9000), (1024, 33, 1, 4),
              (600, 700, 1500, 1504)]


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", LOSS_SIZES)
def test_loss(size, bit):
    from binarybrain_amd import ops
    inputs, channels, frames, pitch = size
    x, values, W, b, label, weight, weight_sum = loss_case(1, inputs, channels, frames, bit, pitch)
    call = (lambda *a, **k: ops.bit_loss_dense_softmax_cross_entropy(*a, pitch, **k)) if bit else ops.loss_dense_softmax_cross_entropy
    give = dict(weight=dev(weight), weight_sum=weight_sum)
    W64, b64 = W.astype(np.float64), b.astype(np.float64)
    want, dz, want_dx, want_dW, want_db = exact_loss(values, W64, b64, label[0, :frames], weight[0, :frames].astype(np.float64), weight_sum)
    z = W64 @ values + b64[:, None]
    z_bound = product_bound(W64, values) + 4 * U * (np.abs(z) + np.abs(b64)[:, None])
    dz_off = loss_bounds(values, W64, b64, dz, weight[0, :frames].astype(np.float64), weight_sum, z_bound)
    loss, dx, dW, db = call(dev(x), dev(W), dev(b), dev(label), frames, **give)
    top = np.abs(z).max(0)
    near(host(loss)[0, :frames], want, weight[0, :frames] * (2 * z_bound.max(0) + 48 * U * (1 + top)) + 8 * U * np.abs(want) + 1e-300, "loss")
    near(host(dx)[:, :frames], want_dx, product_bound(W64.T, dz) + np.abs(W64.T) @ dz_off + 1e-300, "dx")
    near(host(dW), want_dW, product_bound(dz, values.T) + dz_off @ np.abs(values.T) + 1e-300, "dW")
    near(host(db), want_db, product_bound(dz, np.ones((frames, 1)))[:, 0] + dz_off.sum(1) + 1e-300, "db")
    assert np.linalg.norm(host(dx)[:, :frames] - want_dx) <= 2e-5 * np.linalg.norm(want_dx)
    # the loss alone is the same; gradients are added to what is there
    alone = call(dev(x), dev(W), dev(b), dev(label), frames, want_gradients=False, **give)
    assert alone[1] is None and alone[2] is None and np.array_equal(host(alone[0])[:, :frames], host(loss)[:, :frames])
    there = [dev(np.ones(W.shape, np.float32)), dev(np.ones(channels, np.float32))]
    call(dev(x), dev(W), dev(b), dev(label), frames, dW=there[0], db=there[1], want_dx=False, **give)
    assert np.all(np.abs(host(there[0]) - 1 - host(dW)) <= 2 * U * (1 + np.abs(host(dW)))) and np.all(np.abs(host(there[1]) - 1 - host(db)) <= 2 * U * (1 + np.abs(host(db))))


def test_loss_of_nothing():
    """no frame counts: zeros, whatever the frames hold"""
    from binarybrain_amd import ops
    for inputs, channels, frames in ((20, 30, 40), (600, 530, 1100)):
        x = np.full((inputs, frames), np.nan, np.float32)
        W = np.ones((channels, inputs), np.float32)
        out = ops.loss_dense_softmax_cross_entropy(dev(x), dev(W), None, dev(np.full((1, frames), -5, np.int32)), frames)
        assert all(not host(t).any() for t in (out[0][:, :frames], out[2], out[3])) and not host(out[1])[:, :frames].any()


def test_channels_that_are_closed():
    """a bias of minus infinity closes a channel: no probability, no gradient"""
    from binarybrain_amd import ops
    for inputs, channels, frames in ((20, 90, 40), (600, 1030, 1100)):
        rng, x, values, W, b = layer(6, inputs, channels, frames, False, frames)
        closed = np.zeros(channels, bool)
        closed[10:80] = True                                  # whole tiles among them
        b[closed] = -np.inf
        label = rng.integers(0, 10, (1, frames)).astype(np.int32)
        loss, dx, dW, db = ops.loss_dense_softmax_cross_entropy(dev(x), dev(W), dev(b), dev(label), frames)
        keep = ~closed
        at = np.cumsum(keep) - 1
        want, dz, want_dx, want_dW, want_db = exact_loss(values, W[keep].astype(np.float64), b[keep].astype(np.float64), at[label[0]], np.ones(frames), float(frames))
        assert not host(dW)[closed].any() and not host(db)[closed].any()
        assert np.linalg.norm(host(dW)[keep] - want_dW) <= 1e-6 * np.linalg.norm(want_dW) and np.linalg.norm(host(dx) - want_dx) <= 1e-6 * np.linalg.norm(want_dx)
        assert np.linalg.norm(host(loss)[0] - want) <= 1e-6 * np.linalg.norm(want)


def test_loss_of_frames_where_everything_is_certain():
    """probabilities of 1 and 0: loss and gradient 0, no overflow from logits in the thousands"""
    from binarybrain_amd import ops
    x, W = np.full((1, 40), 1000.0, np.float32), np.zeros((70, 1), np.float32)
    W[13] = 7.0
    loss, dx, dW, db = ops.loss_dense_softmax_cross_entropy(dev(x), dev(W), None, dev(np.full(40, 13, np.int32)), 40)
    assert not host(loss)[:, :40].any() and not host(dW).any() and not host(db).any() and not host(dx)[:, :40].any()
    loss = ops.loss_dense_softmax_cross_entropy(dev(x), dev(W), None, dev(np.full(40, 14, np.int32)), 40, want_gradients=False)[0]
    assert np.array_equal(host(loss)[0, :40], np.full(40, 7000.0, np.float32))
