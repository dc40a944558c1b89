"""CPU suite: what the entries of dense layers, of the loss on top of one and of clipped gradients refuse, before anything is launched; their workspaces; rules and objects of the host
classes; the machine code of their kernels."""
import ctypes as C
import os
import re
import subprocess

import pytest

import test_isa as isa
from binarybrain_amd import capi
from binarybrain_amd.build import LIB_PATH
from binarybrain_amd.capi import BbhipError

P = C.c_void_p(1 << 20)             # aligned, and never looked at: every call here is refused
ODD = C.c_void_p((1 << 20) + 16)
MUCH = 1 << 50
NAN, INF = float("nan"), float("inf")


def refused(name, *args):
    lib = capi.lib()
    assert getattr(lib, "bbhip_" + name)(*args) != 0, name
    return lib.bbhip_GetLastErrorString().decode()


# (sizes that need a workspace)
def forward(x=P, y=P, W=P, b=P, r=P, act=0, i=2048, o=1024, f=512, xs=512, ys=512, rs=512, work=P, size=MUCH, bits=False):
    return (x, y, W, b, r) + (() if bits else (act,)) + (i, o, f, xs, ys, rs, work, size, None)


SIZES = [dict(i=0), dict(o=-1), dict(f=0), dict(i=(1 << 24) + 1), dict(o=(1 << 24) + 1), dict(f=(1 << 25) + 1, xs=1 << 30, ys=1 << 30, rs=1 << 30)]


@pytest.mark.parametrize("what", SIZES + [dict(x=None), dict(y=None), dict(W=None), dict(xs=15), dict(ys=15), dict(rs=511), dict(xs=(33 << 20) + 1), dict(rs=(33 << 20) + 1), dict(work=None),
                                          dict(work=ODD), dict(size=4096)])
def test_forward_refuses(what):
    for name in ("fp32", "bit_fp32", "fp32_bit", "bit_bit"):
        assert "DenseAffine_Forward" in refused(name + "_DenseAffine_Forward", *forward(bits=name.endswith("_bit"), **what))
    for act in (-1, 4):
        assert "activation" in refused("fp32_DenseAffine_Forward", *forward(act=act))


def backward(x=P, dy=P, y=P, W=P, dx=P, dW=P, db=P, dr=P, act=1, add=0, i=2048, o=1024, f=512, xs=512, dxs=512, s=512, work=P, size=MUCH):
    return (x, dy, y, W, dx, dW, db, dr, act, add, i, o, f, xs, dxs, s, work, size, None)


@pytest.mark.parametrize("what", SIZES[:5] + [dict(x=None), dict(dy=None), dict(y=None), dict(W=None), dict(dW=None), dict(dx=None, dW=None, db=None, dr=None), dict(act=4), dict(act=-1),
                                              dict(xs=15), dict(dxs=511), dict(s=511), dict(s=(33 << 20) + 1), dict(work=None), dict(work=ODD), dict(size=4096)])
def test_backward_refuses(what):
    for name in ("fp32", "bit_fp32"):
        assert "DenseAffine_Backward" in refused(name + "_DenseAffine_Backward", *backward(**what))


def loss(x=P, W=P, b=P, label=P, weight=P, dx=P, dW=P, db=P, out=P, ws=1.0, add=0, i=64, c=100, f=512, xs=512, dxs=512, work=P, size=MUCH):
    return (x, W, b, label, weight, dx, dW, db, out, ws, add, i, c, f, xs, dxs, work, size, None)


@pytest.mark.parametrize("what", [dict(i=0), dict(c=0), dict(f=-4), dict(i=(1 << 24) + 1), dict(c=(1 << 24) + 1), dict(f=(1 << 25) + 1), dict(x=None), dict(W=None), dict(label=None), dict(out=None),
                                  dict(dW=None), dict(xs=15), dict(dxs=511), dict(dxs=(33 << 20) + 1), dict(work=None), dict(work=ODD), dict(size=64)])
def test_loss_refuses(what):
    for name in ("fp32", "bit_fp32"):
        assert "LossDenseSoftmaxCrossEntropy" in refused(name + "_LossDenseSoftmaxCrossEntropy", *loss(**what))


def norm(n=3, sizes=P, grads=P, most=1.0, out=P, work=P, size=MUCH):
    return (n, sizes, grads, most, out, work, size, None)


@pytest.mark.parametrize("what", [dict(n=-1), dict(sizes=None), dict(grads=None), dict(most=-1.0), dict(most=NAN), dict(out=None), dict(work=None), dict(work=ODD), dict(size=64)])
def test_norm_refuses(what):
    assert "GradientNorm" in refused("fp32_GradientNorm", *norm(**what)) and "GradientClip" in refused("fp32_GradientClip", *norm(**what))
    n, sizes, grads, most, out, work, size, st = norm(**what)
    assert "OptimizerAdam_Clipped" in refused("fp32_OptimizerAdam_Clipped", n, sizes, P, grads, P, P, 0.1, 0.9, 0.999, most, out, 0, work, size, st)


def test_clipped_step_refuses_missing_tables():
    for missing in range(3):
        tables = [P, P, P]
        tables[missing] = None
        assert "null" in refused("fp32_OptimizerAdam_Clipped", 1, P, tables[0], P, tables[1], tables[2], 0.1, 0.9, 0.999, 1.0, P, 0, P, MUCH, None)


def test_workspaces():
    """sizes that an entry refuses need none; what is held of a loss does not grow with the channels beyond a piece's"""
    lib = capi.lib()
    dense, loss_bytes = lib.bbhip_DenseAffine_WorkspaceBytes, lib.bbhip_LossDenseSoftmaxCrossEntropy_WorkspaceBytes
    assert dense(0, 1, 1) == 0 and dense(1, 1 << 25, 1) == 0 and loss_bytes(1, 0, 1, 1) == 0 and loss_bytes(1, 1, 1 << 26, 1) == 0
    for sizes in ((1, 1, 1), (64, 64, 64), (784, 6144, 1024), (4096, 4096, 8192), (6144, 1024, 65)):
        assert dense(*sizes) % 256 == 0 and loss_bytes(*sizes, 0) % 256 == 0 and loss_bytes(*sizes, 1) >= loss_bytes(*sizes, 0)
    # 2^18 channels x 8192 frames are 8 GiB of logits; a piece's logits, gradient (two ways) and weights (two ways) are 1.5 GiB, the sums of the tiles 128 MiB
    a, b = loss_bytes(1024, 1 << 17, 8192, 1), loss_bytes(1024, 1 << 18, 8192, 1)
    assert b < 2 << 30 and b - a <= 160 << 20
    assert lib.bbhip_GradientNorm_WorkspaceBytes() % 256 == 0


def test_calls_refuse_what_is_not_on_the_device():
    import torch
    from binarybrain_amd import ops
    x, W, b, words, label = torch.zeros(4, 8), torch.zeros(3, 4), torch.zeros(3), torch.zeros((4, 1), dtype=torch.int32), torch.zeros((1, 8), dtype=torch.int32)
    dy = torch.zeros(3, 8)
    for call in (lambda: ops.dense_affine_forward(x, W, b, 8), lambda: ops.bit_dense_affine_forward(words, W, b, 8, 8), lambda: ops.dense_affine_forward_bits(x, W, b, 8),
                 lambda: ops.bit_dense_affine_forward_bits(words, W, b, 8), lambda: ops.dense_affine_backward(x, dy, W, 8), lambda: ops.bit_dense_affine_backward(words, dy, W, 8),
                 lambda: ops.loss_dense_softmax_cross_entropy(x, W, b, label, 8), lambda: ops.bit_loss_dense_softmax_cross_entropy(words, W, b, label, 8, 8),
                 lambda: ops.GradientTable([b]), lambda: ops.AdamState([b], [b])):
        with pytest.raises(BbhipError, match="device tensors|on one device"):
            call()
    with pytest.raises(BbhipError, match="gelu"):
        ops.dense_affine_forward(x, W, b, 8, activation="gelu")


def test_rules_and_objects():
    """tests/cpp/test_dense.cpp --rules: how the products are divided over many sizes, and the host classes' objects"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    exe = os.path.join(root, "tests", "cpp", "test_dense")
    if not os.path.exists(exe):
        from binarybrain_amd.build import build_cpp_tests
        build_cpp_tests()
    res = subprocess.run([exe, "--rules"], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert res.returncode == 0, res.stdout


# ---- machine code: the library holds a code object for each of its translation units ---------------------------------------------------
@pytest.fixture(scope="module")
def code(tmp_path_factory):
    """the code object of the dense layers' unit"""
    tools = [os.path.join(isa.LLVM, t) for t in ("llvm-objcopy", "clang-offload-bundler", "llvm-objdump", "llvm-readelf")]
    if not os.path.exists(LIB_PATH) or not all(os.path.exists(t) for t in tools):
        pytest.skip("needs the built library and the LLVM tools of ROCm")
    at = tmp_path_factory.mktemp("isa")
    fat = str(at / "fat")
    subprocess.run([tools[0], "--dump-section", ".hip_fatbin=" + fat, LIB_PATH, os.devnull], check=True, capture_output=True)
    data, magic = open(fat, "rb").read(), b"__CLANG_OFFLOAD_BUNDLE__"
    starts = [m.start() for m in re.finditer(magic, data)] + [len(data)]
    for k in range(len(starts) - 1):
        part, out = str(at / ("part%d" % k)), str(at / ("code%d.o" % k))
        open(part, "wb").write(data[starts[k]:starts[k + 1]])
        subprocess.run([tools[1], "--unbundle", "--type=o", "--input=" + part, "--output=" + out, "--targets=hipv4-amdgcn-amd-amdhsa--gfx950"], check=True, capture_output=True)
        if b"dense_packed_kernel" in open(out, "rb").read():
            return out
    raise AssertionError("no code object holds the dense layers' kernels")


def test_machine_code(code):
    """no 64-bit shift by the last register, loads to LDS a wait state behind their address; and there are some: the products' stages are such loads"""
    notes = subprocess.run([os.path.join(isa.LLVM, "llvm-readelf"), "--notes", code], check=True, capture_output=True, text=True).stdout
    allocated, name = {}, None
    for line in notes.splitlines():
        m = re.match(r"\s+\.name:\s+(_Z\S+)", line)
        name = m.group(1) if m else name
        m = re.match(r"\s+\.vgpr_count:\s+(\d+)", line)
        if m:
            allocated[name] = int(m.group(1))
        # (no kernel of these keeps registers in memory)
        m = re.match(r"\s+\.private_segment_fixed_size:\s+(\d+)", line)
        assert not m or int(m.group(1)) == 0, name
    text = isa.disassembly_of(code).stdout.read().splitlines()
    assert len(allocated) > 30 and sum("load_lds" in line for line in text) > 50
    assert not isa.shifts_by_the_last_register(text, allocated) and not isa.lds_loads_behind_a_write_of_m0(text)
    assert not any(re.search(r"\bv_pk_(add|mul|fma)_f32", line) for line in text)
