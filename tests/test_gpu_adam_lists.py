"""GPU: the lists that AdamState takes, and the plain step beside one whose gradients are not clipped."""
import numpy as np
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


def test_a_step_that_clips_nothing_is_the_plain_one():
    """of betas that are float32 values"""
    import torch
    from binarybrain_amd import ops
    sizes = [4096, 33, 100_001, 1]
    plain, measured = tensors(1, sizes), tensors(1, sizes)
    grads = tensors(2, sizes)
    betas = dict(beta1=np.float32(0.9), beta2=np.float32(0.999))
    a, b = ops.AdamState(plain, grads, **betas), ops.AdamState(measured, grads, **betas)
    for _ in range(3):
        a.step()
        assert b.step(max_norm=float("inf"))[1].item() == 1.0
        for p, q in zip(plain + a.m + a.v, measured + b.m + b.v):
            assert torch.equal(p, q)
