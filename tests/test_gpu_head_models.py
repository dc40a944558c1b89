"""GPU: the operators at the head of a network as a program uses them — the C++ host classes (tests/cpp/test_head.cpp), a run of all of them one after the other,
calls on another stream than the default one, calls that overlap, and steps captured into graphs and replayed."""
import os
import subprocess

import numpy as np
import pytest

import head_reference as ref
from util import dev, host

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32 = np.float32


def test_cpp_classes():
    exe = os.path.join(ROOT, "tests", "cpp", "test_head")
    assert os.path.exists(exe), "tests/cpp/test_head is missing: run __graft_entry__.build()"
    res = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert res.returncode == 0, res.stdout


class Head:
    """buffers of one head, and its step: layer norm -> the student's logits; a teacher's kept logits -> distillation -> layer norm's gradients; a draw"""

    def __init__(self, seed, C, P, F, k):
        import torch
        rng = np.random.default_rng(seed)
        self.C, self.P, self.F, self.k = C, P, F, k
        S = (F + 3) // 4 * 4
        rows = lambda n, scale=1.0: dev((scale * rng.standard_normal((n, S))).astype(F32))
        self.x, self.teacher = rows(C * P), rows(C * P, 3.0)
        self.gamma, self.beta = dev((1 + 0.1 * rng.standard_normal(C * P)).astype(F32)), dev(rng.standard_normal(C * P).astype(F32))
        self.dgamma, self.dbeta = torch.zeros(C * P, device="cuda"), torch.zeros(C * P, device="cuda")
        self.u = dev(rng.random((P, S)).astype(F32))
        self.out = {}

    def step(self):
        from binarybrain_amd import ops
        C, P, F, k = self.C, self.P, self.F, self.k
        self.dgamma.zero_(); self.dbeta.zero_()
        y, mean, rstd = ops.layer_normalization_forward(self.x, self.gamma, self.beta, F)
        index, logit = ops.top_logits(self.teacher, k, C, P, F)
        dy, loss = ops.loss_distillation(y, index, logit, C, P, F, temperature=2.0)
        dx, _, _ = ops.layer_normalization_backward(self.x, dy, self.gamma, mean, rstd, F, dgamma=self.dgamma, dbeta=self.dbeta)
        category, share = ops.categorical_sampling(y, self.u, C, P, F, temperature=0.8, top_size=k, top_p=0.9, min_p=0.01)
        self.out = dict(y=y, index=index, logit=logit, dy=dy, loss=loss, dx=dx, category=category, share=share)

    def results(self):
        got = {n: host(t)[:, :self.F].copy() for n, t in self.out.items()}
        return dict(got, dgamma=host(self.dgamma).copy(), dbeta=host(self.dbeta).copy())


def equal(a, b):
    return [n for n in a if not np.array_equal(a[n], b[n])] == []


SIZES = [(10, 1, 64, 4), (12, 5, 33, 6), (700, 1, 130, 40), (9000, 1, 6, 50), (5000, 1, 300, 20)]


@pytest.mark.parametrize("size", SIZES)
def test_a_head_step(size):
    """each operator's output is the next one's input; checked against 64 bits along the way, from what the operator itself was given"""
    import torch
    head = Head(3, *size)
    C, P, F, k = size
    head.step()
    torch.cuda.synchronize()
    got = head.results()
    cols = lambda a, rows: a.reshape(rows, P * F)
    x, gamma, beta = host(head.x)[:, :F], host(head.gamma), host(head.beta)
    wy, mean, rstd = ref.layer_norm(x, gamma, beta, 1e-5)
    assert np.abs(got["y"] - wy).max() < 5e-5                                   # a hundred roundings of values up to 6
    wi, wv = ref.top_logits(cols(host(head.teacher)[:, :F], C), k)
    assert np.array_equal(cols(got["index"], k), wi) and np.array_equal(cols(got["logit"], k), wv)
    wdy, wloss = ref.distillation(cols(got["y"], C), wi, wv, np.ones(P * F), 2.0, P * F)
    assert np.abs(cols(got["dy"], C) - wdy).max() < 400 * ref.U * 2.0 / (P * F)
    assert np.abs(cols(got["loss"], 1)[0] - wloss).max() < 4 * 400 * ref.U * 30   # T^2, logits up to 15 over T, log of the channels
    wdx, wdg, wdb = ref.layer_norm_backward(x, got["dy"], gamma, mean.astype(F32), rstd.astype(F32))
    scale = np.abs(got["dy"]).max() * 2
    assert np.abs(got["dx"] - wdx).max() < 2e-5 * scale * rstd.max()
    assert np.abs(got["dgamma"] - wdg).max() < 2e-5 * scale * 6 * F and np.abs(got["dbeta"] - wdb).max() < 2e-5 * scale * F
    wc, ws = ref.sampling(cols(got["y"], C), host(head.u)[:, :F].reshape(-1), 0.8, k, 0.9, 0.01)
    assert np.array_equal(cols(got["category"], 1)[0], wc) and np.abs(cols(got["share"], 1)[0] - ws).max() < 2 * ref.U


@pytest.mark.parametrize("size", SIZES)
def test_the_same_bits_every_time(size):
    import torch
    head = Head(4, *size)
    head.step(); torch.cuda.synchronize()
    first = head.results()
    for _ in range(3):
        head.step(); torch.cuda.synchronize()
        assert equal(head.results(), first)


@pytest.mark.parametrize("size", SIZES)
def test_padding_is_left_alone(size):
    """what lies behind the frames of given buffers is not written, and of results only if they are the call's own"""
    import torch
    C, P, F, k = size
    head = Head(5, *size)
    for t in (head.x, head.teacher, head.u):
        t[:, F:] = -77.0
    head.step(); torch.cuda.synchronize()
    for t in (head.x, head.teacher, head.u):
        assert torch.all(t[:, F:] == -77.0)
    # through the C ABI: an output buffer of the caller's keeps its padding, too
    from binarybrain_amd import capi
    y = torch.full_like(head.x, -5.0)
    work = torch.empty(max(int(capi.lib().bbhip_LayerNormalization_WorkspaceBytes(C * P, F)), 1), dtype=torch.uint8, device="cuda")
    p = capi.ptr
    capi.check(capi.lib().bbhip_fp32_LayerNormalization_Forward(p(head.x), p(y), p(head.gamma), p(head.beta), None, None, 1e-5, C * P, F, y.shape[1], y.shape[1], p(work),
                                                               work.numel(), capi.stream_ptr()))
    torch.cuda.synchronize()
    assert torch.all(y[:, F:] == -5.0) and np.array_equal(host(y)[:, :F], head.results()["y"])
    # in place
    x = head.x.clone()
    capi.check(capi.lib().bbhip_fp32_LayerNormalization_Forward(p(x), p(x), p(head.gamma), p(head.beta), None, None, 1e-5, C * P, F, x.shape[1], x.shape[1], p(work),
                                                               work.numel(), capi.stream_ptr()))
    torch.cuda.synchronize()
    assert np.array_equal(host(x)[:, :F], head.results()["y"]) and torch.all(x[:, F:] == -77.0)


def test_streams_that_overlap():
    """two heads at once, each on a stream of its own: their workspaces are their own"""
    import torch
    heads = [Head(6 + i, 9000, 1, 40, 50) for i in range(2)]
    torch.cuda.synchronize()
    for h in heads:
        h.step()
    torch.cuda.synchronize()
    want = [h.results() for h in heads]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for h, s in zip(heads, streams):
            with torch.cuda.stream(s):
                h.step()
    torch.cuda.synchronize()
    assert all(equal(h.results(), w) for h, w in zip(heads, want))


@pytest.mark.parametrize("size", SIZES)
def test_replays_equal_eager(size):
    """two captured steps, replayed in turn and at once on two streams, with eager work between: every replay equals the eager step on the same inputs"""
    import torch
    heads = [Head(8 + i, *size) for i in range(2)]
    for h in heads:
        h.step()
    torch.cuda.synchronize()
    graphs = []
    for h in heads:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            h.step()
        graphs.append((g, dict(h.out)))
    eager = [Head(8 + i, *size) for i in range(2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    rng = np.random.default_rng(30)
    for k in range(4):
        for h, e in zip(heads, eager):
            for name in ("x", "teacher", "u"):
                t = rng.standard_normal(getattr(h, name).shape).astype(F32) if name != "u" else rng.random(h.u.shape).astype(F32)
                getattr(h, name).copy_(dev(t)); getattr(e, name).copy_(dev(t))
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            if k % 2:
                with torch.cuda.stream(s):
                    g.replay()
            else:
                g.replay()
        torch.cuda.synchronize()
        for h, e, (_, out) in zip(heads, eager, graphs):
            e.step()
            torch.cuda.synchronize()
            h.out = out
            assert equal(h.results(), e.results()), k
