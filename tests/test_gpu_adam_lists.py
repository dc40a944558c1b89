"""GPU: the lists that AdamState takes."""
import pytest

pytestmark = pytest.mark.gpu


def tensors(seed, sizes):
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return [torch.randn(n, generator=gen, device="cuda") for n in sizes]


def test_lists_of_unequal_length():
    """too few gradients or moments are refused as everything else is; gradients behind the last parameter's are not looked at"""
    import torch
    from binarybrain_amd import ops
    from binarybrain_amd.capi import BbhipError
    params, grads = tensors(1, [40, 70]), tensors(2, [40, 70])
    for given in (dict(grads=grads[:1]), dict(grads=[]), dict(grads=grads, m=tensors(3, [40])), dict(grads=grads, v=tensors(3, [40, 70, 5]))):
        with pytest.raises(BbhipError, match="2 parameters"):
            ops.AdamState(params, **given)
    for max_norm in (None, 0.5):
        more, same = [p.clone() for p in params], [p.clone() for p in params]
        a, b = ops.AdamState(more, grads + tensors(4, [9])), ops.AdamState(same, grads)
        for _ in range(2):
            a.step(max_norm=max_norm)
            b.step(max_norm=max_norm)
        assert all(torch.equal(p, q) for p, q in zip(more, same)) and len(a.grads) == 3
