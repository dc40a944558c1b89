"""GPU: the operators at the head of a network where two of their paths have to agree, at the ends of their ranges, and in the variants that only large calls take.
Tolerances are those of test_gpu_head_operators.py unless a test derives its own."""
import numpy as np
import pytest

import head_reference as ref
from head_reference import U
from test_gpu_head_operators import F32, check_distill, check_norm, check_norm_backward, columns, distill_case, logits_of, near, ops, padded, same_values  # noqa: F401 (ops: the fixture)
from util import dev, host

pytestmark = pytest.mark.gpu


# ---- lists that name a channel again with minus infinity -------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(30, 40, 12), (33, 40, 12), (700, 40, 12), (700, 37, 12), (33, 24, 200), (5000, 260, 200)])
def test_distillation_of_lists_padded_with_minus_infinity(ops, shape):
    """an entry of minus infinity has no share, whatever else its channel is named for: before, behind and between entries that have one"""
    C, F, k = shape
    rng = np.random.default_rng(C + F)
    y, index, z, w = distill_case(rng, C, F, min(k, C))
    if k > C:
        index = np.concatenate([index, rng.integers(0, C, (k - C, F)).astype(np.int32)])
        z = np.concatenate([z, rng.standard_normal((k - C, F)).astype(F32)])
    none = F32(-np.inf)
    index[1, 0] = 0; index[6:, 0] = 0; z[6:, 0] = none                       # the usual padding, and channel 0 is listed
    index[0, 1] = index[3, 1]; z[0, 1] = none                                # before
    index[9, 2] = index[3, 2]; z[9, 2] = none                                # behind
    index[[2, 5, 8], 3] = index[4, 3]; z[[2, 5, 8], 3] = none                # several
    index[[7, 9], 4] = index[2, 4]; z[9, 4] = none                           # two shares and one without
    index[1:, 5] = index[0, 5]; z[1:, 5] = none                              # nothing but one channel
    index[:, 6] = C - 1; z[:-1, 6] = none                                    # the last entry alone
    few = rng.integers(0, C, 5)
    some = np.arange(F) >= F // 2                                            # five channels all over, half of the entries without a share
    index[:, some] = few[rng.integers(0, 5, (k, some.sum()))]
    z[:, some] = np.where(rng.random((k, some.sum())) < 0.5, none, z[:, some])
    z[0, some] = 1.0
    call = lambda: [host(a) for a in ops.loss_distillation(dev(y), dev(index), dev(z), C, 1, F, temperature=1.5, weight=dev(w[None]), weight_sum=5.0)]
    dy, loss = call()
    check_distill(y, index, z, w, 1.5, 5.0, dy, loss[0])
    for _ in range(3):
        again = call()
        assert np.array_equal(again[0], dy) and np.array_equal(again[1], loss)


# ---- layer normalisation of far values -------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("nodes", [100, 1000, 20000])                         # one launch, one launch, two
@pytest.mark.parametrize("frames", [9, 12])                                  # rows that start on 4 bytes, on 16
@pytest.mark.parametrize("kind", [(1e20, 0.01, 1e-5), (1e30, 0.01, 1e-5), (-1e30, 1.0, 1e-5), (1e18, 1.0, 1e-5), (1e-20, 0.01, 0.0), (1e-25, 1.0, 0.0), (1e-3, 1.0, 1e-5)])
def test_layer_norm_of_far_values(ops, nodes, frames, kind):
    """values whose squares leave the range of float32, upwards and (with eps 0) downwards: statistics and y are those of the definition all the same.
    A rounding of the mean is at most U of the largest value, 100 of them 6e-6 of it: with deviations of 1 % of the values 6e-4 of the deviation, which check_norm counts."""
    scale, spread, eps = kind
    rng = np.random.default_rng(nodes + frames)
    x = (scale * (1.0 + spread * rng.standard_normal((nodes, frames)))).astype(F32)
    gamma, beta = (1 + 0.3 * rng.standard_normal(nodes)).astype(F32), rng.standard_normal(nodes).astype(F32)
    y, mean, rstd = ops.layer_normalization_forward(dev(x), dev(gamma), dev(beta), frames, eps=eps)
    check_norm(x, gamma, beta, host(y), host(mean), host(rstd), *ref.layer_norm(x, gamma, beta, float(F32(eps))))
    assert np.all(np.abs(host(rstd) / ref.layer_norm(x, gamma, beta, float(F32(eps)))[2] - 1) < 1e-4)
    # what the forward pass leaves serves the backward pass
    dy = rng.standard_normal((nodes, frames)).astype(F32)
    dx, dgamma, dbeta = ops.layer_normalization_backward(dev(x), dev(dy), dev(gamma), mean, rstd, frames)
    check_norm_backward(x, dy, gamma, host(mean), host(rstd), host(dx), host(dgamma), host(dbeta), *ref.layer_norm_backward(x, dy, gamma, host(mean), host(rstd)))


@pytest.mark.parametrize("nodes", [300, 20000])
@pytest.mark.parametrize("frames", [40, 41])
def test_layer_norm_of_frames_that_are_not_finite(ops, nodes, frames):
    """rstd of a frame that holds an infinity or what is not a number is not a number, in one launch and in two, and so is all of its y; the others keep their bits"""
    rng = np.random.default_rng(nodes)
    x = rng.standard_normal((nodes, frames)).astype(F32)
    clean = [host(a) for a in ops.layer_normalization_forward(dev(x), None, None, frames)]
    x[17, 3], x[250, 21], x[0, 22], x[nodes - 1, 30] = np.nan, np.inf, -np.inf, np.nan
    y, mean, rstd = (host(a) for a in ops.layer_normalization_forward(dev(x), None, None, frames))
    touched = np.isin(np.arange(frames), (3, 21, 22, 30))
    assert np.all(np.isnan(rstd[touched])) and not np.any(np.isfinite(mean[touched])) and np.all(np.isnan(y[:, touched]))
    assert np.array_equal(y[:, ~touched], clean[0][:, ~touched]) and np.array_equal(mean[~touched], clean[1][~touched]) and np.array_equal(rstd[~touched], clean[2][~touched])


@pytest.mark.parametrize("nodes", [100, 300, 3000, 20000])
@pytest.mark.parametrize("frames", [40, 41])
@pytest.mark.parametrize("eps", [1e-5, 0.0])
def test_layer_norm_of_far_frames_among_others(ops, nodes, frames, eps):
    """far values in all rows of a frame, in half of them and in one: that frame's statistics follow the definition, every other frame keeps its bits"""
    rng = np.random.default_rng(nodes)
    x = rng.standard_normal((nodes, frames)).astype(F32)
    gamma, beta = (1 + 0.3 * rng.standard_normal(nodes)).astype(F32), rng.standard_normal(nodes).astype(F32)
    clean = [host(a) for a in ops.layer_normalization_forward(dev(x), dev(gamma), dev(beta), frames, eps=eps)]
    x[:, 5] = 1e25 * (np.arange(nodes) - nodes / 3)
    x[nodes // 2:, 6] = 1e28
    x[nodes - 2, 7] = -1e29
    x[:, 18] *= F32(1e-25)
    y, mean, rstd = (host(a) for a in ops.layer_normalization_forward(dev(x), dev(gamma), dev(beta), frames, eps=eps))
    wy, wmean, wrstd = ref.layer_norm(x, gamma, beta, float(F32(eps)))
    check_norm(x, gamma, beta, y, mean, rstd, wy, wmean, wrstd)
    assert np.all(np.abs(rstd / wrstd - 1) < 1e-4)
    same = ~np.isin(np.arange(frames), (5, 6, 7, 18))
    assert np.array_equal(y[:, same], clean[0][:, same]) and np.array_equal(mean[same], clean[1][same]) and np.array_equal(rstd[same], clean[2][same])


# ---- near the ends of the ranges -------------------------------------------------------------------------------------------------------
def test_layer_norm_of_more_than_2_28_frames(ops):
    """what only the form with rows on 16 bytes serves; dgamma against sums in 64 bits, 2^18 tiles of 256 frames in a chain"""
    import torch
    nodes, F = 2, (1 << 28) + 8
    gen = torch.Generator(device="cuda"); gen.manual_seed(2)
    x, dy = torch.randn((nodes, F), generator=gen, device="cuda"), torch.randn((nodes, F), generator=gen, device="cuda")
    gamma, beta = np.array([1.5, 0.5], F32), np.array([-1.0, 2.0], F32)
    y, mean, rstd = ops.layer_normalization_forward(x, dev(gamma), dev(beta), F)
    dx, dgamma, dbeta = ops.layer_normalization_backward(x, dy, dev(gamma), mean, rstd, F)
    for part in (slice(0, 2000), slice((1 << 28) - 1000, F)):
        v, d, m, r = host(x[:, part]), host(dy[:, part]), host(mean[part]), host(rstd[part])
        check_norm(v, gamma, beta, host(y[:, part]), m, r, *ref.layer_norm(v, gamma, beta, float(F32(1e-5))))
        wdx, wdg, wdb = ref.layer_norm_backward(v, d, gamma, m, r)
        check_norm_backward(v, d, gamma, m, r, host(dx[:, part]), wdg, wdb, wdx, wdg, wdb)
    for n in range(nodes):
        each = dy[n].double() * ((x[n].double() - mean.double()) * rstd.double())
        near(float(dgamma[n]), float(each.sum()), (2 ** 18 + 200) * U * float(each.abs().sum()), "dgamma")
        near(float(dbeta[n]), float(dy[n].double().sum()), (2 ** 18 + 200) * U * float(dy[n].abs().double().sum()), "dbeta")


def test_logits_of_many_places(ops):
    """33 channels: 2^25 places of distillation, 2^27 - 16 of selection in fours"""
    import torch
    C, k = 33, 2
    gen = torch.Generator(device="cuda"); gen.manual_seed(3)
    F = 1 << 25
    y = torch.randn((C, F), generator=gen, device="cuda")
    index, logit = ops.top_logits(y, k, C, 1, F)
    dy, loss = ops.loss_distillation(y, index, logit, C, 1, F, temperature=2.0, weight_sum=3.0)
    for part in (slice(0, 500), slice(F // 2 - 250, F // 2 + 250), slice(F - 500, F)):
        v = host(y[:, part])
        wi, wv = ref.top_logits(v, k)
        assert np.array_equal(host(index[:, part]), wi) and np.array_equal(host(logit[:, part]), wv)
        check_distill(v, wi, wv, np.ones(500, F32), 2.0, 3.0, host(dy[:, part]), host(loss[:, part])[0])
    del y, dy, loss, index, logit
    F = (1 << 27) - 16
    y, u = torch.randn((C, F), generator=gen, device="cuda"), torch.rand((1, F), generator=gen, device="cuda")
    category, share = ops.categorical_sampling(y, u, C, 1, F, top_size=k)
    for part in (slice(0, 500), slice(F // 2 - 250, F // 2 + 250), slice(F - 500, F)):
        wc, ws = ref.sampling(host(y[:, part]), host(u[0, part]), 1.0, k, 1.0, 0.0)
        assert np.array_equal(host(category[0, part]), wc)
        near(host(share[0, part]), ws, 2 * U * ws, "share")


# ---- defaults --------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("C", [1, 10, 49, 50, 51, 300])
def test_sampling_with_the_defaults(ops, C):
    """50 of the largest logits, or all of fewer channels"""
    rng = np.random.default_rng(C)
    y, u = (3 * rng.standard_normal((C, 40))).astype(F32), rng.random(40).astype(F32)
    category, share = ops.categorical_sampling(dev(y), dev(u[None]), C, 1, 40)
    wc, ws = ref.sampling(y, u, 1.0, min(C, 50), 1.0, 0.0)
    assert np.array_equal(host(category)[0], wc)
    near(host(share)[0], ws, 2 * U * ws, "share")


# ---- variants that only large calls take (tests/cpp/test_head.cpp --rules holds that these shapes take them) ----------------------------
@pytest.mark.parametrize("shape", [(1025, 4097, 4100), (1100, 4099, 4100), (4096, 8190, 8192), (257, 4097, 4097), (1024, 8191, 8191),      # 16 rows per thread, of four frames and of one
                                   (4097, 8190, 8192), (3000, 8193, 8196), (1025, 8191, 8191)])                                            # just beyond: two launches
def test_layer_norm_of_long_columns(ops, shape):
    nodes, F, stride = shape
    rng = np.random.default_rng(nodes)
    x = (rng.standard_normal((nodes, F), dtype=F32) * rng.uniform(0.5, 3, F).astype(F32) + rng.uniform(-4, 4, F).astype(F32))
    gamma, beta = (1 + 0.3 * rng.standard_normal(nodes)).astype(F32), rng.standard_normal(nodes).astype(F32)
    given = dev(padded(x, stride))
    y, mean, rstd = ops.layer_normalization_forward(given, dev(gamma), dev(beta), F)
    got, mean, rstd = host(y)[:, :F], host(mean), host(rstd)
    for at in range(0, F, 1024):                                             # (in parts: 64-bit copies of the whole are large)
        part = slice(at, at + 1024)
        check_norm(x[:, part], gamma, beta, got[:, part], mean[part], rstd[part], *ref.layer_norm(x[:, part], gamma, beta, float(F32(1e-5))))
    # in place, without statistics: the same bits, and the padding stays
    from binarybrain_amd import capi
    import torch
    work = torch.empty(max(int(capi.lib().bbhip_LayerNormalization_WorkspaceBytes(nodes, F)), 1), dtype=torch.uint8, device="cuda")
    p, g, b = capi.ptr, dev(gamma), dev(beta)
    capi.check(capi.lib().bbhip_fp32_LayerNormalization_Forward(p(given), p(given), p(g), p(b), None, None, 1e-5, nodes, F, stride, stride, p(work), work.numel(), capi.stream_ptr()))
    torch.cuda.synchronize()
    again = host(given)
    assert np.array_equal(again[:, :F], got) and np.all(np.isnan(again[:, F:]))


SCAN_SHAPES = [
    # channels, frames, stride, k: four units of a row side by side, of four frames where the pitch allows
    (3100, 2050, 2052, 64), (3100, 2050, 2052, 200), (10000, 1030, 1032, 100),       # several slabs and the join, bounds from 256 and from 512 groups
    (2000, 1025, 1025, 40), (3200, 2050, 2051, 120), (2500, 2050, 2051, 7),          # one frame per thread; one slab in several rounds
]


def sorted_logits(y, k):
    """the operator's order by a stable sort of 64-bit numbers: infinity for what is not a number, the next below for infinity"""
    v = y.astype(np.float64) + 0.0
    v = np.where(np.isnan(v), np.inf, np.where(v == np.inf, 1e308, v))
    order = np.argsort(-np.ascontiguousarray(v.T), axis=1, kind="stable")[:, :k].T.astype(np.int32)
    return order, np.take_along_axis(y, order, 0)


@pytest.mark.parametrize("shape", SCAN_SHAPES)
@pytest.mark.parametrize("kind", ["random", "equal", "constant", "ascending", "descending", "special"])
def test_top_logits_of_large_calls(ops, shape, kind):
    C, F, stride, k = shape
    y = logits_of(kind, np.random.default_rng(C + F), (C, F))
    index, logit = ops.top_logits(dev(padded(y, stride, np.inf)), k, C, 1, F)
    wi, wv = sorted_logits(y, k)
    assert np.array_equal(host(index)[:, :F], wi) and same_values(host(logit)[:, :F], wv)


@pytest.mark.parametrize("shape", [SCAN_SHAPES[1], SCAN_SHAPES[2], SCAN_SHAPES[3], SCAN_SHAPES[4]])
@pytest.mark.parametrize("rule", [(0.7, 0.9, 0.0), (2.0, 1.0, 0.02)])
def test_sampling_of_large_calls(ops, shape, rule):
    C, F, stride, k = shape
    t, top_p, min_p = rule
    for kind in ("equal", "ascending", "special"):
        rng = np.random.default_rng(C + 5 * F)
        y, u = logits_of(kind, rng, (C, F)), rng.random(F).astype(F32)
        category, share = ops.categorical_sampling(dev(padded(y, stride, np.inf)), dev(padded(u[None], stride)), C, 1, F, temperature=t, top_size=k, top_p=top_p, min_p=min_p)
        wi, wv = sorted_logits(y, k)
        wc, ws = ref.sampling(wv, u, t, k, top_p, min_p)                     # (of the k largest in their order: positions, then channels)
        wc = np.where(wc >= 0, np.take_along_axis(wi, np.maximum(wc, 0)[None], 0)[0], -1)
        assert np.array_equal(host(category)[0, :F], wc), kind
        near(host(share)[0, :F], ws, 2 * U * ws, kind)


# ---- a mean that is large against the deviation ----------------------------------------------------------------------------------------
@pytest.mark.parametrize("nodes", [1000, 3000])                              # one launch, two
@pytest.mark.parametrize("stride", [72, 70])                                 # four frames at a time, one
@pytest.mark.parametrize("offset", [1e3, 1e4, 1e5])
def test_layer_norm_of_a_large_mean_by_its_roundings(ops, nodes, stride, offset):
    """The longest way of a value into the mean has 25 roundings of at most U * offset: eight rows summed and scaled (5.4: their partial sums are k * offset, over 8), then a
    merge each for a second batch, 3 wavefronts, 12 slabs of a thread and 3 wavefronts again; in one launch 3 rows, up to 4 lane steps, 16 wavefronts and a quotient.
    A group of n rows whose mean is off by e <= 25 U offset adds e^2 to the variance, and to the sum of squares between groups at most 2 e / sqrt(n) of unit deviation: over the
    levels (8 rows 3.8, 16 rows 3.2, 64 rows 1.6 + 5.3, the rest 2) no more than 16 U offset, half of that in rstd."""
    rng = np.random.default_rng(nodes)
    F, c = 70, offset * U
    x = (offset + rng.standard_normal((nodes, F))).astype(F32)
    y, mean, rstd = ops.layer_normalization_forward(dev(padded(x, stride)), None, None, F)
    one, zero = np.ones(nodes, F32), np.zeros(nodes, F32)
    wy, wmean, wrstd = ref.layer_norm(x, one, zero, float(F32(1e-5)))
    near(host(mean), wmean, 25 * c * 1.01, "mean")                           # (the largest value is a little above the offset)
    rel = 8 * c + 0.5 * (25 * c) ** 2 + 128 * U
    near(host(rstd), wrstd, wrstd * rel, "rstd")
    near(host(y)[:, :F], wy, wrstd * 26 * c * (1 + rel) + np.abs(wy) * (rel + 4 * U), "y")


# ---- workspaces ------------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(40, 1, 8, 3), (700, 1, 24, 9), (1000, 1, 1, 50), (2000, 3, 13, 40), (5000, 1, 300, 20), (9000, 1, 68, 100), (20000, 1, 5, 50), (3000, 1, 1000, 4)])
def test_workspaces_of_the_size_asked_for(ops, shape):
    """each entry does with the bytes that its ..._WorkspaceBytes names, from rows on 16 bytes and from rows that are not, and leaves what lies behind them"""
    import torch
    from binarybrain_amd import capi
    C, P, F, k = shape
    lib, p, nodes = capi.lib(), capi.ptr, C * P
    rng = np.random.default_rng(C + F)
    S = (F + 3) // 4 * 4 + 4

    def rows(a, off):                                                        # [rows, S], `off` floats behind a start on 256 bytes
        t = torch.zeros(a.shape[0] * S + off, dtype=torch.float32 if a.dtype == F32 else torch.int32, device="cuda")[off:].view(a.shape[0], S)
        t[:, :F] = dev(a)
        return t

    def run(name, size, *args):
        work = torch.full((size + 512,), 0xa5, dtype=torch.uint8, device="cuda")
        capi.check(getattr(lib, "bbhip_" + name)(*args, p(work) if size else None, size, capi.stream_ptr()))
        torch.cuda.synchronize()
        assert bool((work[size:] == 0xa5).all()), name

    x, dy = rng.standard_normal((nodes, F)).astype(F32), rng.standard_normal((nodes, F)).astype(F32)
    line = lambda n: torch.ones(n, device="cuda")
    got = []
    for off in (0, 1):
        a, d, out = rows(x, off), rows(dy, off), rows(np.zeros_like(x), off)
        bits = torch.zeros((nodes, (F + 31) // 32), dtype=torch.int32, device="cuda")
        mean, rstd, g, b = line(F + 4)[off:], line(F + 4)[off:], line(nodes), line(nodes)
        norm = lib.bbhip_LayerNormalization_WorkspaceBytes(nodes, F)
        run("fp32_LayerNormalization_Forward", norm, p(a), p(out), p(g), p(b), p(mean), p(rstd), 1e-5, nodes, F, S, S)
        y = host(out)[:, :F].copy()
        run("bit_fp32_LayerNormalization_Forward", norm, p(bits), p(out), p(g), p(b), p(line(F + 4)[off:]), p(line(F + 4)[off:]), 1e-5, nodes, F, bits.shape[1], S)
        dg, db = line(nodes), line(nodes)
        run("fp32_LayerNormalization_Backward", norm, p(a), p(d), p(out), p(g), p(mean), p(rstd), p(dg), p(db), 0, nodes, F, S, S)
        dx = host(out)[:, :F].copy()
        run("bit_fp32_LayerNormalization_Backward", norm, p(bits), p(d), p(out), p(g), p(mean), p(rstd), p(dg), p(db), 0, nodes, F, bits.shape[1], S)
        top = lib.bbhip_TopLogits_WorkspaceBytes(k, P, C, F)
        index, logit = rows(np.zeros((k * P, F), np.int32), off), rows(np.zeros((k * P, F), F32), off)
        run("fp32_TopLogits", top, p(a), p(index), p(logit), k, P, C, F, S, S)
        loss, category, u = rows(np.zeros((P, F), F32), off), rows(np.zeros((P, F), np.int32), off), rows(rng.random((P, F)).astype(F32) if not off else got[0][5], off)
        run("fp32_LossDistillation", lib.bbhip_LossDistillation_WorkspaceBytes(P, C, F), p(a), p(index), p(logit), None, p(out), p(loss), 2.0, 1.0, k, P, C, F, S, S)
        run("fp32_CategoricalSampling", top, p(a), p(u), p(category), None, 1.0, k, 0.9, 0.0, P, C, F, S)
        got.append((y, dx, host(index)[:, :F], host(logit)[:, :F], host(category)[:, :F], host(u)[:, :F].copy(), host(out)[:, :F], host(loss)[:, :F]))
    one = np.ones(nodes, F32)
    wy, _, wrstd = ref.layer_norm(x, one, one, float(F32(1e-5)))
    for y, dx, index, logit, category, _, dy_of, loss in got:
        near(y, wy, 5e-5, "y")                                               # (132 U of values up to 5, and the mean's 100 U times 5)
        wi, wv = ref.top_logits(columns(x, C, P, F), k)
        assert np.array_equal(columns(index, k, P, F), wi) and np.array_equal(columns(logit, k, P, F), wv)
        check_distill(columns(x, C, P, F), wi, wv, np.ones(P * F, F32), 2.0, 1.0, columns(dy_of, C, P, F), columns(loss, 1, P, F)[0])
    assert np.array_equal(got[0][4], got[1][4])
    near(got[0][1], got[1][1], 5e-5 * wrstd.max() * (1 + np.abs(dy).max()), "dx")


@pytest.mark.parametrize("shape", [(300, 41, 44), (1024, 1000, 1000), (5000, 130, 131), (64, 5000, 5000)])
def test_layer_norm_backward_in_place(ops, shape):
    """dx may be dy: the same bits, and the padding stays"""
    import torch
    from binarybrain_amd import capi
    nodes, F, S = shape
    rng = np.random.default_rng(nodes)
    x, dy = dev(rng.standard_normal((nodes, S)).astype(F32)), dev(padded(rng.standard_normal((nodes, F)).astype(F32), S))
    gamma, line = dev(rng.standard_normal(nodes).astype(F32)), lambda: torch.zeros(nodes, device="cuda")
    _, mean, rstd = ops.layer_normalization_forward(x, gamma, None, F)
    dx, dgamma, dbeta = ops.layer_normalization_backward(x, dy, gamma, mean, rstd, F)
    size, p, dg, db = capi.lib().bbhip_LayerNormalization_WorkspaceBytes(nodes, F), capi.ptr, line(), line()
    work = torch.empty(size, dtype=torch.uint8, device="cuda")
    capi.check(capi.lib().bbhip_fp32_LayerNormalization_Backward(p(x), p(dy), p(dy), p(gamma), p(mean), p(rstd), p(dg), p(db), 0, nodes, F, S, S, p(work), size, capi.stream_ptr()))
    torch.cuda.synchronize()
    assert np.array_equal(host(dy)[:, :F], host(dx)[:, :F]) and np.all(np.isnan(host(dy)[:, F:]))
    assert np.array_equal(host(dg), host(dgamma)) and np.array_equal(host(db), host(dbeta))
