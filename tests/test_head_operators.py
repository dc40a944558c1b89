"""CPU suite: what the operators at the head of a network refuse, before anything is launched, and the sizes of their workspaces."""
import ctypes as C

import pytest

from binarybrain_amd import capi
from binarybrain_amd.capi import BbhipError

P = C.c_void_p(1 << 20)             # aligned, and never looked at: every call here is refused
MIB = 1 << 20


def refused(name, *args):
    lib = capi.lib()
    assert getattr(lib, "bbhip_" + name)(*args) != 0, name
    return lib.bbhip_GetLastErrorString().decode()


# (sizes that need a workspace: short columns and few channels go without one)
def norm(x=P, y=P, gamma=P, beta=P, mean=P, rstd=P, eps=1e-5, nodes=20000, frames=16, xs=16, ys=16, work=P, size=MIB):
    return (x, y, gamma, beta, mean, rstd, eps, nodes, frames, xs, ys, work, size, None)


@pytest.mark.parametrize("what", [dict(x=None), dict(y=None), dict(nodes=0), dict(nodes=-3), dict(frames=0), dict(xs=15), dict(ys=15), dict(eps=-1.0), dict(eps=float("nan")),
                                  dict(work=None), dict(size=16), dict(work=C.c_void_p((1 << 20) + 16)), dict(nodes=1 << 20, frames=(1 << 30) + 3, xs=(1 << 30) + 3, ys=(1 << 30) + 3), dict(nodes=(1 << 30) + 1)])
def test_layer_norm_forward_refuses(what):
    assert "LayerNormalization_Forward" in refused("fp32_LayerNormalization_Forward", *norm(**what))
    if what not in (dict(xs=15),):
        refused("bit_fp32_LayerNormalization_Forward", *norm(**what))


def test_bits_count_words():
    assert "stride" in refused("bit_fp32_LayerNormalization_Forward", *norm(frames=33, xs=1, ys=64))


def norm_backward(x=P, dy=P, dx=P, gamma=P, mean=P, rstd=P, dgamma=P, dbeta=P, add=0, nodes=8, frames=16, xs=16, s=16, work=P, size=MIB):
    return (x, dy, dx, gamma, mean, rstd, dgamma, dbeta, add, nodes, frames, xs, s, work, size, None)


@pytest.mark.parametrize("what", [dict(x=None), dict(dy=None), dict(dx=None), dict(mean=None), dict(rstd=None), dict(nodes=0), dict(frames=-1), dict(xs=3), dict(s=15),
                                  dict(work=None), dict(size=64), dict(work=C.c_void_p((1 << 20) + 4))])
def test_layer_norm_backward_refuses(what):
    assert "LayerNormalization_Backward" in refused("fp32_LayerNormalization_Backward", *norm_backward(**what))
    if what != dict(xs=3):
        refused("bit_fp32_LayerNormalization_Backward", *norm_backward(**what))


def top(y=P, index=P, logit=P, k=4, pix=1, ch=10, frames=16, s=16, ls=16, work=P, size=MIB):
    return (y, index, logit, k, pix, ch, frames, s, ls, work, size, None)


@pytest.mark.parametrize("what", [dict(y=None), dict(index=None), dict(logit=None), dict(k=0), dict(k=11), dict(k=257, ch=1000), dict(pix=0), dict(ch=-1), dict(frames=0), dict(s=15),
                                  dict(ls=15), dict(pix=1 << 16, ch=1 << 16), dict(ch=(1 << 30) + 1), dict(pix=1 << 27), dict(ch=100000, frames=1, work=C.c_void_p((1 << 20) + 64)), dict(ch=100000, frames=1, work=None), dict(ch=100000, frames=1, size=8)])
def test_top_logits_refuses(what):
    assert "TopLogits" in refused("fp32_TopLogits", *top(**what))


def distill(y=P, index=P, logit=P, weight=P, dy=P, loss=P, t=1.0, ws=1.0, k=4, pix=1, ch=100, frames=16, s=16, ls=16, work=P, size=MIB):
    return (y, index, logit, weight, dy, loss, t, ws, k, pix, ch, frames, s, ls, work, size, None)


@pytest.mark.parametrize("what", [dict(y=None), dict(index=None), dict(logit=None), dict(dy=None), dict(loss=None), dict(t=0.0), dict(t=-1.0), dict(t=float("inf")), dict(t=float("nan")), dict(t=1e-30), dict(t=1e30),
                                  dict(k=0), dict(k=257), dict(pix=-1), dict(ch=0), dict(frames=0), dict(s=8), dict(ls=8), dict(work=None), dict(size=1)])
def test_distillation_refuses(what):
    assert "LossDistillation" in refused("fp32_LossDistillation", *distill(**what))


def sample(y=P, u=P, category=P, share=P, t=1.0, k=4, top_p=1.0, min_p=0.0, pix=1, ch=10, frames=16, s=16, work=P, size=MIB):
    return (y, u, category, share, t, k, top_p, min_p, pix, ch, frames, s, work, size, None)


@pytest.mark.parametrize("what", [dict(y=None), dict(u=None), dict(category=None), dict(t=0.0), dict(t=float("nan")), dict(k=0), dict(k=11), dict(k=300, ch=400), dict(top_p=0.0),
                                  dict(top_p=1.5), dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=1.1), dict(pix=0), dict(frames=0), dict(s=15)])
def test_sampling_refuses(what):
    assert "CategoricalSampling" in refused("fp32_CategoricalSampling", *sample(**what))


def test_workspaces():
    """sizes that an entry refuses need none; larger problems need no less than an entry asks for"""
    lib = capi.lib()
    assert lib.bbhip_LayerNormalization_WorkspaceBytes(0, 5) == 0 and lib.bbhip_LayerNormalization_WorkspaceBytes(5, -1) == 0
    assert lib.bbhip_TopLogits_WorkspaceBytes(0, 1, 5, 5) == 0 and lib.bbhip_TopLogits_WorkspaceBytes(257, 1, 500, 5) == 0
    assert lib.bbhip_LossDistillation_WorkspaceBytes(1, 0, 5) == 0
    for nodes, frames in ((1, 1), (1000, 1), (4096, 8192), (3, 100000)):
        size = lib.bbhip_LayerNormalization_WorkspaceBytes(nodes, frames)
        assert size >= 0 and size % 256 == 0
    assert lib.bbhip_TopLogits_WorkspaceBytes(50, 1, 32768, 1) % 256 == 0


def test_calls_refuse_what_is_not_on_the_device():
    import torch
    from binarybrain_amd import ops
    x, line, rows = torch.zeros(4, 8), torch.zeros(4), torch.zeros((4, 8), dtype=torch.int32)
    for call in (lambda: ops.layer_normalization_forward(x, line, line, 8), lambda: ops.bit_layer_normalization_forward(rows, line, line, 8, 8),
                 lambda: ops.layer_normalization_backward(x, x, line, line, line, 8), lambda: ops.bit_layer_normalization_backward(rows, x, line, line, line, 8),
                 lambda: ops.top_logits(x, 2, 4, 1, 8), lambda: ops.loss_distillation(x, rows, x, 4, 1, 8), lambda: ops.categorical_sampling(x, x, 4, 1, 8, top_size=2)):
        with pytest.raises(BbhipError, match="device tensors"):
            call()
    with pytest.raises(TypeError):
        ops.top_logits([1, 2], 2, 4, 1, 8)


def test_rules_and_objects():
    """tests/cpp/test_head.cpp --rules: how the column operators divide their work over many sizes, and the host classes' objects"""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = os.path.join(root, "tests", "cpp", "test_head")
    if not os.path.exists(exe):
        from binarybrain_amd.build import build_cpp_tests
        build_cpp_tests()
    res = subprocess.run([exe, "--rules"], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert res.returncode == 0, res.stdout
