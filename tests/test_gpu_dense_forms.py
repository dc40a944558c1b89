"""Every form of a dense product (straight or packed, tiles of each size, a k axis shared or not, one or four rows for few frames) against 64 bits: the cases of the other sizes, at sizes whose
rule takes that form."""
import numpy as np
import pytest

import test_gpu_dense as cases
from dense_reference import loss as exact_loss

pytestmark = pytest.mark.gpu

# (inputs, outputs, frames, pitch)
FORWARD = [(6144, 100, 65, 66), (2048, 10, 64, 64), (1024, 128, 128, 131), (70, 5200, 3, 4), (64, 5121, 8, 8), (301, 6001, 1, 1),        # straight: shared k axes, four rows for few frames
           (1100, 640, 1300, 1301), (300, 2600, 2500, 2500), (64, 9000, 1400, 1408), (145, 21806, 548, 548)]                              # packed: shared, small, large, middle tiles
BACKWARD = [(64, 64, 1030, 1031), (2049, 33, 70, 70), (300, 4100, 70, 72), (640, 530, 1100, 1101), (784, 1500, 1024, 1024), (300, 2600, 1100, 1100), (6193, 995, 128, 128)]


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", FORWARD)
def test_forward(size, bit):
    cases.test_forward(size, bit)


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", BACKWARD)
def test_backward(size, bit):
    cases.test_backward(size, bit)


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", [(2048, 40, 70, 96), (1100, 640, 1300, 1312), (300, 2600, 2500, 2528), (30, 5300, 5, 32)])
def test_forward_to_bits(size, bit):
    cases.test_forward_to_bits(size, bit)


@pytest.mark.parametrize("size", [(2048, 40, 60), (1100, 640, 1300), (300, 2600, 2500), (120, 5300, 40)])
def test_special_values(size):
    cases.test_special_values(size)


@pytest.mark.parametrize("size", [(2048, 40, 60), (1100, 640, 1300), (300, 2600, 2500)])
def test_scales_of_rows(size):
    cases.test_scales_of_rows(size)


@pytest.mark.parametrize("bit", [False, True])
@pytest.mark.parametrize("size", [(2048, 10, 64, 64), (8192, 40, 100, 101), (1600, 640, 700, 704), (300, 1500, 1030, 1031)])
def test_loss(size, bit):
    cases.test_loss(size, bit)


def test_loss_of_nothing():
    from binarybrain_amd import ops
    for inputs, channels, frames in ((2048, 10, 40), (700, 900, 1100)):
        x = np.full((inputs, frames), np.nan, np.float32)
        W = np.ones((channels, inputs), np.float32)
        out = ops.loss_dense_softmax_cross_entropy(cases.dev(x), cases.dev(W), None, cases.dev(np.full((1, frames), -5, np.int32)), frames)
        assert all(not cases.host(t).any() for t in (out[0][:, :frames], out[2], out[3])) and not cases.host(out[1])[:, :frames].any()


def test_channels_that_are_closed():
    """whole tiles and the label's neighbours without a probability, where the logits' k axis is shared"""
    from binarybrain_amd import ops
    for inputs, channels, frames in ((2048, 70, 40), (1600, 640, 700)):
        rng, x, values, W, b = cases.layer(6, inputs, channels, frames, False, frames)
        closed = np.zeros(channels, bool)
        closed[5:69] = True
        b[closed] = -np.inf
        label = rng.integers(0, 5, (1, frames)).astype(np.int32)
        loss, dx, dW, db = ops.loss_dense_softmax_cross_entropy(cases.dev(x), cases.dev(W), cases.dev(b), cases.dev(label), frames)
        keep = ~closed
        want, dz, want_dx, want_dW, want_db = exact_loss(values, W[keep].astype(np.float64), b[keep].astype(np.float64), label[0], np.ones(frames), float(frames))
        assert not cases.host(dW)[closed].any() and not cases.host(db)[closed].any()
        # (labels lie ahead of the closed channels, so their numbers stay)
        for got, exact in ((cases.host(dW)[keep], want_dW), (cases.host(db)[keep], want_db), (cases.host(dx), want_dx), (cases.host(loss)[0], want)):
            assert np.linalg.norm(got - exact) <= 1e-6 * np.linalg.norm(exact)
