"""GPU parity of the norm of a list of gradients, of clipping, and of the Adam step with clipped gradients."""
import numpy as np
import pytest

from dense_reference import U

pytestmark = pytest.mark.gpu


def tensors(seed, sizes, off=()):
    """one tensor per size, float32 on the device; those of `off` start four bytes behind a multiple of 16"""
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    out = []
    for k, n in enumerate(sizes):
        t = torch.randn(n + 1, generator=gen, device="cuda") * 10.0 ** (k % 7 - 3)
        out.append(t[1:] if k in off else t[:n])
    return out


def exact_norm(ts):
    return float(np.sqrt(sum((t.cpu().numpy().astype(np.float64) ** 2).sum() for t in ts)))


LISTS = [([1], ()), ([4096], ()), ([4095, 4096, 4097], (1,)), ([0, 3, 0, 8192, 1], (3,)), ([5] * 700 + [100000] + [1] * 300, (2, 700)), ([3_000_001, 70, 5_000_000], (0,)),
         ([4096 * 1025, 1, 4096 * 3], ()), ([17] * 256, ()), ([17] * 257, ())]


@pytest.mark.parametrize("which", range(len(LISTS)))
def test_norm_and_clip(which):
    from binarybrain_amd import ops
    sizes, off = LISTS[which]
    ts = tensors(which, sizes, off)
    exact = exact_norm(ts)
    table = ops.GradientTable(ts)
    norm, scale = table.norm().tolist()
    assert abs(norm - exact) <= 2 * U * exact and scale == 1.0
    again = table.norm(exact / 3)
    assert again[0].item() == norm and abs(again[1].item() - 1 / 3) <= 4 * U
    before = [t.clone() for t in ts]
    assert table.clip_(exact * 1.5).tolist() == [norm, 1.0] and all(bool((a == b).all()) for a, b in zip(ts, before))
    clipped = table.clip_(exact / 3)
    assert clipped.tolist() == again.tolist()
    assert all(bool((a == b * clipped[1]).all()) for a, b in zip(ts, before))
    assert abs(table.norm()[0].item() - exact / 3) <= 8 * U * exact
    assert table.clip_(0.0)[1].item() == 0.0 and not any(bool(t.any()) for t in ts) and table.clip_(0.0).tolist() == [0.0, 1.0]


def test_values_whose_squares_leave_float32():
    import torch
    from binarybrain_amd import ops
    for v in (1e30, 1e-30, 3e38, 1e-44):
        t = torch.full((5000,), v, device="cuda")
        want = exact_norm([t])
        norm, scale = ops.GradientTable([t]).norm(1.0).tolist()
        # (2^-150: half a step of the numbers below 2^-126, where a relative one does not hold)
        assert (norm == np.inf if want > 3.4e38 else abs(norm - want) <= 2 * U * want + 2.0 ** -150) and abs(scale - min(1.0, 1.0 / want)) <= 2 * U


def test_values_that_are_not_finite():
    import torch
    from binarybrain_amd import ops
    a, b = torch.ones(10, device="cuda"), torch.ones(5000, device="cuda")
    b[77] = np.inf
    assert ops.GradientTable([a, b]).clip_(2.0).tolist() == [np.inf, 0.0]
    assert not a.any() and int(b.isnan().sum()) == 1 and int((b == 0).sum()) == 4999
    b = torch.ones(5000, device="cuda")
    b[78] = np.nan
    norm, scale = ops.GradientTable([b]).clip_(2.0).tolist()
    assert np.isnan(norm) and scale == 1.0 and int((b == 1).sum()) == 4999


@pytest.mark.parametrize("share", [0.3, 2.0])
@pytest.mark.parametrize("update", [False, True])
def test_adam_with_clipped_gradients(share, update):
    """the bits of the plain step on gradients that were scaled before"""
    import torch
    from binarybrain_amd import ops
    sizes, off = [4096, 33, 100_001, 1], (1,)
    params, grads = tensors(1, sizes, off), tensors(2, sizes, off)
    plain_params, plain_grads = [p.clone() for p in params], [g.clone() for g in grads]
    before = [g.clone() for g in grads]
    max_norm = share * exact_norm(grads)
    betas = dict(beta1=0.875, beta2=0.9921875)              # (floats: 1 - beta is the same in 32 and 64 bits)
    clipped, plain = ops.AdamState(params, grads, **betas), ops.AdamState(plain_params, plain_grads, **betas)
    for step in range(3):
        norm = (clipped.update if update else clipped.step)(max_norm=max_norm)
        scale = ops.GradientTable(plain_grads).clip_(max_norm)
        assert norm.tolist() == scale.tolist() and (norm[1].item() < 1) == (share < 1 and bool(norm[0] > 0))
        plain.step()
        for p, q in zip(params + clipped.m + clipped.v, plain_params + plain.m + plain.v):
            assert torch.equal(p, q)
        if update:
            assert not any(bool(g.any()) for g in grads)
            for g, h, b in zip(grads, plain_grads, before):
                g.copy_(b * (step + 1)); h.copy_(b * (step + 1))
        else:
            assert all(torch.equal(g, b) for g, b in zip(grads, before))
            for h, b in zip(plain_grads, before):
                h.copy_(b)


def test_lists_that_are_refused():
    import torch
    from binarybrain_amd import ops
    from binarybrain_amd.capi import BbhipError
    t = torch.ones(8, device="cuda")
    for bad in ([t, t], [], [t.cpu()], [t.double()], [torch.ones((4, 4), device="cuda").t()]):
        with pytest.raises(BbhipError):
            ops.GradientTable(bad)
    for bad in (-1.0, float("nan")):
        with pytest.raises(BbhipError, match="max_norm"):
            ops.GradientTable([t]).norm(bad)


def test_a_clipped_step_refuses_a_tensor_twice():
    import torch
    from binarybrain_amd import ops
    from binarybrain_amd.capi import BbhipError
    p, q, g, h = (torch.ones(8, device="cuda") for _ in range(4))
    for params, grads in (([p, p], [g, h]), ([p, q], [g, g]), ([p], [p])):
        for step in ("step", "update"):
            with pytest.raises(BbhipError, match="twice"):
                getattr(ops.AdamState(params, grads), step)(max_norm=1.0)
