"""GPU: the operators at the head of a network where two of their paths have to agree, at the ends of their ranges, and in the variants that only large calls take.
Tolerances are those of test_gpu_head_operators.py unless a test derives its own."""
import numpy as np
import pytest

import head_reference as ref
from test_gpu_head_operators import F32, as_rows, check_distill, columns, distill_case, ops  # noqa: F401 (ops: the fixture)
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
