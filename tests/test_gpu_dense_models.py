"""GPU: dense layers, the loss on top of one and clipped gradients as a program uses them — the C++ host classes (tests/cpp/test_dense.cpp), a training step of all of them one after the
other, workspaces of exactly the size asked for, padding, calls on other streams, calls that overlap, and steps captured into graphs and replayed."""
import os
import subprocess

import numpy as np
import pytest

from dense_reference import U, activated, bits_of, loss as exact_loss, product_bound, through
from util import dev, host

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
F32 = np.float32


def test_cpp_classes():
    exe = os.path.join(ROOT, "tests", "cpp", "test_dense")
    assert os.path.exists(exe), "tests/cpp/test_dense is missing: run __graft_entry__.build()"
    res = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=300)
    assert res.returncode == 0, res.stdout


class Net:
    """x (fp32 or bits) -> dense, sigmoid -> dense with a residual, hard tanh -> the loss of a dense head; clipped Adam step"""

    def __init__(self, seed, inputs, hidden, channels, F, bit):
        import torch
        from binarybrain_amd import ops
        rng = np.random.default_rng(seed)
        self.F, self.bit, self.S = F, bit, (F + 63) // 64 * 64
        normal = lambda *shape, scale=1.0: dev((scale * rng.standard_normal(shape)).astype(F32))
        self.x = dev(rng.integers(-2 ** 31, 2 ** 31, (inputs, self.S // 32)).astype(np.int32)) if bit else normal(inputs, self.S)
        sizes = [(hidden, inputs), (hidden, hidden), (channels, hidden)]
        self.W = [normal(o, i, scale=2.0 / np.sqrt(i)) for o, i in sizes]
        self.b = [normal(o, scale=0.1) for o, _ in sizes]
        self.dW, self.db = [torch.zeros_like(w) for w in self.W], [torch.zeros_like(b) for b in self.b]
        label = rng.integers(0, channels, (1, F)).astype(np.int32)
        label[0, 3::7] = -1
        self.label, self.weight = dev(label), dev((rng.random((1, F)) + 0.5).astype(F32))
        self.weight_sum = float((host(self.weight) * (label >= 0)).sum())
        self.adam = ops.AdamState(self.W + self.b, self.dW + self.db, 0.01, 0.875, 0.9921875)
        self.out = {}

    def step(self, update=True):
        from binarybrain_amd import ops
        F, W, b = self.F, self.W, self.b
        for g in self.dW + self.db:
            g.zero_()
        h1 = ops.bit_dense_affine_forward(self.x, W[0], b[0], F, self.S, activation="sigmoid") if self.bit else ops.dense_affine_forward(self.x, W[0], b[0], F, activation="sigmoid")
        h2 = ops.dense_affine_forward(h1, W[1], b[1], F, activation="hard_tanh", residual=h1)
        loss, dh2, _, _ = ops.loss_dense_softmax_cross_entropy(h2, W[2], b[2], self.label, F, weight=self.weight, weight_sum=self.weight_sum, dW=self.dW[2], db=self.db[2])
        dh1, _, _, dr = ops.dense_affine_backward(h1, dh2, W[1], F, activation="hard_tanh", y=h2, dW=self.dW[1], db=self.db[1], want_dr=True)
        both = ops.vector_add_ex(dh1, dr)
        back = ops.bit_dense_affine_backward if self.bit else ops.dense_affine_backward
        dx, _, _, _ = back(self.x, both, W[0], F, activation="sigmoid", y=h1, dW=self.dW[0], db=self.db[0])
        self.out = dict(h1=h1, h2=h2, loss=loss, dh2=dh2, both=both, dx=dx)
        if update:
            self.out["norm"] = self.adam.step(max_norm=0.5)

    def results(self):
        got = {n: host(t)[:, :self.F].copy() if t.dim() == 2 else host(t).copy() for n, t in self.out.items()}
        for k in range(3):
            got.update({"W%d" % k: host(self.W[k]).copy(), "b%d" % k: host(self.b[k]).copy(), "dW%d" % k: host(self.dW[k]).copy(), "db%d" % k: host(self.db[k]).copy()})
        return got


def differ(a, b):
    return [n for n in a if not np.array_equal(a[n], b[n])]


SIZES = [(20, 24, 10, 40, False), (70, 33, 7, 65, True), (300, 520, 700, 1100, False), (640, 544, 1030, 1300, True), (9, 40, 3000, 5, False)]


@pytest.mark.parametrize("size", SIZES)
def test_a_training_step(size):
    """each operator's output is the next one's input; checked against 64 bits along the way, from what the operator itself was given"""
    import torch
    net = Net(3, *size)
    F, bit = net.F, net.bit
    W, b = [host(w).astype(np.float64) for w in net.W], [host(v).astype(np.float64) for v in net.b]
    net.step(update=False)
    torch.cuda.synchronize()
    got = net.results()
    x = bits_of(host(net.x), F) if bit else host(net.x)[:, :F].astype(np.float64)
    near = lambda name, want, bound: np.testing.assert_array_less(np.abs(got[name] - want), bound + 1e-30, err_msg=name)
    z = W[0] @ x + b[0][:, None]
    near("h1", activated(z, "sigmoid"), product_bound(W[0], x) + 8 * U * (1 + np.abs(z)))
    h1, h2 = got["h1"].astype(np.float64), got["h2"].astype(np.float64)
    z = W[1] @ h1 + b[1][:, None] + h1
    near("h2", activated(z, "hard_tanh"), product_bound(W[1], h1) + 8 * U * (1 + np.abs(z)))
    weight = host(net.weight)[0].astype(np.float64)
    want, dz, want_dh, want_dW, want_db = exact_loss(h2, W[2], b[2], host(net.label)[0], weight, net.weight_sum)
    assert np.linalg.norm(got["loss"][0] - want) <= 2e-6 * np.linalg.norm(want)
    for name, exact in (("dh2", want_dh), ("dW2", want_dW), ("db2", want_db)):
        assert np.linalg.norm(got[name] - exact) <= 2e-6 * np.linalg.norm(exact), name
    dh2 = got["dh2"].astype(np.float64)
    dz = through(dh2, h2, "hard_tanh")
    near("dW1", dz @ h1.T, product_bound(dz, h1.T))
    near("db1", dz.sum(1), product_bound(dz, np.ones((F, 1)))[:, 0])
    near("both", W[1].T @ dz + dz, product_bound(W[1].T, dz) + 2 * U * (np.abs(dz) + np.abs(W[1].T @ dz)))
    dz = through(got["both"].astype(np.float64), h1, "sigmoid")
    slack = 4 * U * np.abs(dz)
    near("dx", W[0].T @ dz, product_bound(W[0].T, dz) + np.abs(W[0].T) @ slack)
    near("dW0", dz @ x.T, product_bound(dz, x.T) + slack @ np.abs(x.T))


@pytest.mark.parametrize("size", SIZES)
def test_the_same_bits_every_time(size):
    import torch
    a, b = Net(4, *size), Net(4, *size)
    for _ in range(3):
        a.step(); torch.cuda.synchronize()
        b.step(); torch.cuda.synchronize()
        assert not differ(a.results(), b.results())


def test_streams_that_overlap():
    """two nets at once, each on a stream of its own: their workspaces are their own"""
    import torch
    want, nets = [Net(6 + i, 300, 520, 700, 1100, False) for i in range(2)], [Net(6 + i, 300, 520, 700, 1100, False) for i in range(2)]
    torch.cuda.synchronize()
    for w in want:
        for _ in range(4):
            w.step()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    torch.cuda.synchronize()
    for _ in range(4):
        for n, s in zip(nets, streams):
            with torch.cuda.stream(s):
                n.step()
    torch.cuda.synchronize()
    for n, w in zip(nets, want):
        assert not differ(n.results(), w.results())


@pytest.mark.parametrize("size", SIZES)
def test_replays_equal_eager(size):
    """two captured steps, replayed in turn and at once on two streams, with eager work between: every replay equals the eager step on the same inputs"""
    import torch
    nets, eager = [Net(8 + i, *size) for i in range(2)], [Net(8 + i, *size) for i in range(2)]
    for n in nets:
        n.step(update=False)
    torch.cuda.synchronize()
    graphs = []
    for n in nets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            n.step(update=False)
        graphs.append((g, dict(n.out)))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    rng = np.random.default_rng(30)
    for k in range(4):
        for n, e in zip(nets, eager):
            t = rng.integers(-2 ** 31, 2 ** 31, n.x.shape).astype(np.int32) if n.bit else rng.standard_normal(n.x.shape).astype(F32)
            n.x.copy_(dev(t)); e.x.copy_(dev(t))
        torch.cuda.synchronize()
        for (g, _), s in zip(graphs, streams):
            if k % 2:
                with torch.cuda.stream(s):
                    g.replay()
            else:
                g.replay()
        torch.cuda.synchronize()
        for n, e, (_, out) in zip(nets, eager, graphs):
            e.step(update=False)
            torch.cuda.synchronize()
            n.out = out
            assert not differ(n.results(), e.results()), k


def test_a_clipped_step_in_a_graph():
    import torch
    from binarybrain_amd import ops
    grads = [torch.randn(n, device="cuda") for n in (5000, 3, 100_000)]
    table = ops.GradientTable(grads)
    table.clip_(1.0); torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = table.clip_(1.0)
    for k in range(4):
        fresh = [torch.randn(t.shape, device="cuda") * (0.001 if k == 2 else 1.0) for t in grads]
        for t, f in zip(grads, fresh):
            t.copy_(f)
        g.replay(); torch.cuda.synchronize()
        other = [f.clone() for f in fresh]
        want = ops.GradientTable(other).clip_(1.0)
        assert out.tolist() == want.tolist() and all(torch.equal(a, b) for a, b in zip(grads, other))


@pytest.mark.parametrize("size", [(40, 50, 33), (2100, 30, 70), (700, 600, 1300), (4, 3, 9000)])
@pytest.mark.parametrize("off", [0, 1])
def test_workspaces_and_padding(size, off):
    """through the C ABI: workspaces of exactly the size asked for, filled with anything, nothing written behind them; rows behind the frames keep what they hold; buffers off 16 bytes and pitches of their own"""
    import torch
    from binarybrain_amd import capi
    inputs, outputs, F = size
    rng = np.random.default_rng(1)
    lib, p = capi.lib(), capi.ptr
    S = {"x": F + 1 + off, "y": F + 5, "r": F + 2, "dx": F + 7}

    def rows(a, pitch):
        t = torch.full((a.shape[0] * pitch + off,), -77.0, device="cuda")[off:].view(a.shape[0], pitch)
        t[:, :F] = dev(a)
        return t

    def run(name, size, *args):
        work = torch.full((size + 512,), 0xff, dtype=torch.uint8, device="cuda")
        capi.check(getattr(lib, "bbhip_" + name)(*args, p(work) if size else None, size, capi.stream_ptr()))
        torch.cuda.synchronize()
        assert bool((work[size:] == 0xff).all()), name

    normal = lambda *shape: rng.standard_normal(shape).astype(F32)
    xv, rv, dyv, Wv = normal(inputs, F), normal(outputs, F), normal(outputs, F), normal(outputs, inputs)
    x, r, dy, W, b = rows(xv, S["x"]), rows(rv, S["r"]), rows(dyv, S["y"]), dev(Wv), dev(np.ones(outputs, F32))
    y, dx, dr = rows(np.zeros((outputs, F), F32), S["y"]), rows(np.zeros((inputs, F), F32), S["dx"]), rows(np.zeros((outputs, F), F32), S["y"])
    n = lib.bbhip_DenseAffine_WorkspaceBytes(inputs, outputs, F)
    run("fp32_DenseAffine_Forward", n, p(x), p(y), p(W), p(b), p(r), 0, inputs, outputs, F, S["x"], S["y"], S["r"])
    x64, W64, dz = xv.astype(np.float64), Wv.astype(np.float64), dyv.astype(np.float64)
    z = W64 @ x64 + 1 + rv
    assert np.all(np.abs(host(y)[:, :F] - z) <= product_bound(W64, x64) + 8 * U * (np.abs(z) + 1 + np.abs(rv)))
    # the residual's buffer as the output's
    run("fp32_DenseAffine_Forward", n, p(x), p(r), p(W), p(b), p(r), 0, inputs, outputs, F, S["x"], S["r"], S["r"])
    assert np.array_equal(host(r)[:, :F], host(y)[:, :F])
    dW, db = torch.zeros_like(W), torch.zeros_like(b)
    run("fp32_DenseAffine_Backward", n, p(x), p(dy), None, p(W), p(dx), p(dW), p(db), p(dr), 0, 0, inputs, outputs, F, S["x"], S["dx"], S["y"])
    assert np.all(np.abs(host(dx)[:, :F] - W64.T @ dz) <= product_bound(W64.T, dz)) and np.all(np.abs(host(dW) - dz @ x64.T) <= product_bound(dz, x64.T))
    assert np.array_equal(host(dr)[:, :F], dyv)
    label, loss = dev(rng.integers(0, outputs, F + off).astype(np.int32))[off:], rows(np.zeros((1, F), F32), F + 3)
    for gradients in (0, 1):
        run("fp32_LossDenseSoftmaxCrossEntropy", lib.bbhip_LossDenseSoftmaxCrossEntropy_WorkspaceBytes(inputs, outputs, F, gradients), p(x), p(W), p(b), p(label), None,
            p(dx) if gradients else None, p(dW) if gradients else None, p(db) if gradients else None, p(loss), float(F), 0, inputs, outputs, F, S["x"], S["dx"])
        want, _, want_dx, want_dW, want_db = exact_loss(x64, W64, np.ones(outputs), host(label), np.ones(F), float(F))
        assert np.linalg.norm(host(loss)[0, :F] - want) <= 1e-6 * np.linalg.norm(want)
    for t, exact in ((host(dx)[:, :F], want_dx), (host(dW), want_dW), (host(db), want_db)):
        assert np.linalg.norm(t - exact) <= 2e-5 * np.linalg.norm(exact)
    for t in (x, r, dy, y, dx, dr, loss):
        assert bool((t[:, F:] == -77.0).all())


def test_calls_are_refused():
    import torch
    from binarybrain_amd import ops
    from binarybrain_amd.capi import BbhipError
    x, W, b, r = torch.zeros((4, 8), device="cuda"), torch.zeros((3, 4), device="cuda"), torch.zeros(3, device="cuda"), torch.zeros((3, 8), device="cuda")
    label = torch.zeros((1, 8), dtype=torch.int32, device="cuda")
    for call in (lambda: ops.dense_affine_forward(x, W, b, 9), lambda: ops.dense_affine_forward(x, W.t().contiguous(), b, 8), lambda: ops.dense_affine_forward(x, W, b[:2], 8),
                 lambda: ops.dense_affine_forward(x.double(), W, b, 8), lambda: ops.dense_affine_forward(x, W, b, 8, residual=r[:2]), lambda: ops.dense_affine_forward(x, W, b, 8, y_stride=7),
                 lambda: ops.dense_affine_forward(x, W, b, 0), lambda: ops.dense_affine_backward(x, r, W, 8, activation="relu"), lambda: ops.dense_affine_backward(x, r[:2], W, 8),
                 lambda: ops.dense_affine_backward(x, r, W, 8, dW=torch.zeros_like(W)), lambda: ops.dense_affine_backward(x, r, W, 8, want_dx=False, want_weights=False),
                 lambda: ops.loss_dense_softmax_cross_entropy(x, W, b, label.long(), 8, weight_sum=1.0), lambda: ops.loss_dense_softmax_cross_entropy(x, W, b, label[:, :7], 8, weight_sum=1.0),
                 lambda: ops.bit_dense_affine_forward(x, W, b, 8, 8), lambda: ops.AdamState([b], [r])):
        with pytest.raises(BbhipError):
            call()
