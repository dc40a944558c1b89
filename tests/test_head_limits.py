"""CPU suite: the ends of the ranges of the operators at the head of a network.  What a launch cannot hold is refused before the first one, and sizes that one form of an entry
serves have a workspace whatever another form says."""
import ctypes as C

import pytest

from binarybrain_amd import capi
from test_head_operators import P, distill, norm_backward, refused, sample, top

ODD = C.c_void_p((1 << 20) + 4)     # (rows that do not start on 16 bytes: one frame at a time)
MUCH = 1 << 50


@pytest.mark.parametrize("call", [
    ("fp32_LossDistillation", distill(ch=33, frames=1 << 26, s=1 << 26, ls=1 << 26, size=MUCH)),
    ("fp32_LossDistillation", distill(ch=33, pix=1 << 13, frames=1 << 13, s=1 << 13, ls=1 << 13, size=MUCH)),
    ("fp32_LossDistillation", distill(y=ODD, ch=1000, frames=(1 << 26) - 1, s=1 << 26, ls=1 << 26, size=MUCH)),
    ("fp32_TopLogits", top(k=1, ch=33, frames=1 << 27, s=1 << 27, ls=1 << 27, size=MUCH)),
    ("fp32_TopLogits", top(y=ODD, k=1, ch=33, frames=1 << 25, s=1 << 25, ls=1 << 25, size=MUCH)),
    ("fp32_CategoricalSampling", sample(k=1, ch=33, frames=1 << 27, s=1 << 27, size=MUCH)),
    ("fp32_CategoricalSampling", sample(y=ODD, k=1, ch=33, pix=1 << 12, frames=1 << 13, s=1 << 13, size=MUCH)),
    ("fp32_LayerNormalization_Backward", norm_backward(nodes=1 << 30, frames=1, xs=1, s=1, size=MUCH)),
    ("bit_fp32_LayerNormalization_Backward", norm_backward(nodes=1 << 30, frames=1, xs=1, s=1, size=MUCH)),
])
def test_more_threads_than_a_launch_holds(call):
    assert "2^32 threads" in refused(call[0], *call[1])


def test_workspaces_of_large_calls():
    """the form with rows on 16 bytes goes on where the other one ends; 0 where neither goes"""
    lib = capi.lib()
    norm, distillation = lib.bbhip_LayerNormalization_WorkspaceBytes, lib.bbhip_LossDistillation_WorkspaceBytes
    for nodes in (1, 2, 60):
        for frames in ((1 << 28) + 4, 1 << 29, (1 << 30) - 64):
            # sums per frame and, of tiles of 256 frames, per node
            assert norm(nodes, frames) >= 8 * frames + 8 * nodes * (frames // 256)
        assert norm(nodes, (1 << 30) + 4) == 0
    assert norm(1 << 30, 1) >= 64 * 8
    assert distillation(1, 33, 1 << 25) >= 24 << 25 and distillation(1 << 10, 33, 1 << 15) >= 24 << 25
    assert distillation(1, 33, 1 << 26) == 0 and distillation(1 << 20, 33, 1 << 20) == 0
