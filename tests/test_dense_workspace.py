"""The workspace of a dense layer's forward pass alone: what it says (CPU), and that a forward pass takes it and no less (GPU)."""
import numpy as np
import pytest

from binarybrain_amd import capi

SIZES = [(40, 50, 33), (1, 1, 1), (2100, 30, 70), (8192, 300, 5), (700, 600, 1300), (1100, 640, 1300), (4096, 4096, 8192)]


def test_sizes():
    """never more than both passes need, nothing for few frames and for whole straight products, less than half of both where the layer is large and its inputs are packed bits"""
    lib = capi.lib()
    both, forward = lib.bbhip_DenseAffine_WorkspaceBytes, lib.bbhip_DenseAffine_Forward_WorkspaceBytes
    for size in SIZES:
        for bit in (0, 1):
            assert forward(*size, bit) % 256 == 0 and forward(*size, bit) <= both(*size)
    assert forward(40, 50, 33, 0) == forward(8192, 300, 8, 0) == forward(1, 1, 1, 1) == 0
    assert forward(0, 1, 1, 0) == 0 and forward(1, 1 << 25, 1, 0) == 0
    large = (4096, 4096, 8192)
    # 4 bytes of halves per weight and per value, 2 per bit, and 8 for each row and column
    assert forward(*large, 0) == 4 * (4096 * 4096 + 4096 * 8192) + 8 * (4096 + 8192) and forward(*large, 1) == 4 * 4096 * 4096 + 2 * 4096 * 8192 + 8 * 4096 + 4 * 8192
    assert 3 * forward(*large, 1) < both(*large)


@pytest.mark.gpu
@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", SIZES[:-1])
def test_a_forward_pass_takes_it(size, bit):
    import torch
    from binarybrain_amd import ops
    inputs, outputs, frames = size
    lib, p = capi.lib(), capi.ptr
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)
    x = torch.randint(-(1 << 31), 1 << 31, (inputs, frames // 32 + 1), generator=gen, device="cuda", dtype=torch.int64).to(torch.int32) if bit else torch.randn((inputs, frames), generator=gen, device="cuda")
    W, y = torch.randn((outputs, inputs), generator=gen, device="cuda"), torch.empty((outputs, frames), device="cuda")
    n = lib.bbhip_DenseAffine_Forward_WorkspaceBytes(inputs, outputs, frames, int(bit))
    work = torch.full((n + 512,), 0xff, dtype=torch.uint8, device="cuda")
    entry = lib.bbhip_bit_fp32_DenseAffine_Forward if bit else lib.bbhip_fp32_DenseAffine_Forward
    call = lambda size: entry(p(x), p(y), p(W), None, None, 0, inputs, outputs, frames, x.shape[1], frames, 0, p(work) if size else None, size, capi.stream_ptr())
    if n:
        assert call(n - 1) != 0
    capi.check(call(n))
    torch.cuda.synchronize()
    assert bool((work[n:] == 0xff).all())
    want = ops.bit_dense_affine_forward(x, W, None, frames, frames) if bit else ops.dense_affine_forward(x, W, None, frames)
    assert torch.equal(y, want[:, :frames])
