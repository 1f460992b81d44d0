"""The lowest scale of an 8-bit block, max(largest magnitude / 448, 2^-126), at its border: blocks whose largest magnitude is one fp32 number or a
few around 448 * 2^-126, and far below it."""
import pytest
import torch

from block8_util import DEV, TYPES, ULP, check_8_bits

pytestmark = pytest.mark.gpu

BORDER, LEAST = 448 * 2.0 ** -126, 2.0 ** -126


def maxima():
    """fp32 numbers around the border: a step of them there is 2^-141."""
    steps = [0, 1, 2, 3, 10, 100, 600, 1000, 1003, 5000]
    return torch.tensor(sorted({BORDER + d * s * 2.0 ** -141 for s in steps for d in (-1, 1)} | {5.2656e-36, 1e-36, 1e-42, 2.0 ** -149, 1e-35}), device=DEV)


def check_scales(scales, most, off):
    """scales of blocks whose largest magnitude is `most` but for `off` (relative): rounded once, and never under the least one."""
    want = (most.double() / 448).clamp_min(LEAST)
    assert bool((scales >= LEAST).all()), float(scales.min())
    assert bool(((scales.double() - want).abs() <= want * (off + ULP)).all())
    if off == 0:
        assert bool((scales[most.double() <= BORDER] == LEAST).all())


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("cols", [256, 258, 129])
def test_rows(kind, cols):
    from dlprimitives_b200 import capi
    most = maxima().to(TYPES[kind])
    x = torch.zeros(len(most), cols, dtype=TYPES[kind], device=DEV)
    x[:, 128] = -most                                # alone in its block, and beside smaller ones
    x[:, 5], x[:, 100] = most, most / 2
    q, scales = torch.empty(len(most), cols, dtype=TYPES["e4m3"], device=DEV), torch.empty(-(-cols // 128), len(most), device=DEV)
    capi.quantize(x, q, scales)
    check_scales(scales[0], most, 0)
    check_scales(scales[1], most, 0)
    check_8_bits(q, scales.t(), x.double(), 1, 0.0)


@pytest.mark.parametrize("cols", [128, 130])
def test_blocks(cols):
    from dlprimitives_b200 import capi
    most = maxima()
    x = torch.zeros(128 * len(most), cols, device=DEV)
    x[3::128, 77], x[127::128, 0] = most, -most / 4
    q, scales = torch.empty(x.shape, dtype=TYPES["e4m3"], device=DEV), torch.empty(len(most), -(-cols // 128), device=DEV)
    capi.quantize(x, q, scales, block_rows=128)
    check_scales(scales[:, 0], most, 0)
    check_8_bits(q, scales, x.double(), 128, 0.0)


@pytest.mark.parametrize("cols", [128, 127])
def test_norm(cols):
    """The output's magnitude is the weight's here: rows of one value and an eps that is small beside it.  One weight vector a call."""
    from dlprimitives_b200 import capi
    for most in maxima():
        x = torch.ones(1, cols, device=DEV)
        w = torch.zeros(cols, device=DEV)
        w[9] = most
        y, scales = torch.empty(1, cols, dtype=TYPES["e4m3"], device=DEV), torch.empty(1, 1, device=DEV)
        capi.rms_norm(x, w, y, scales=scales, eps=1e-12)
        # the sum of ones is exact; the mean, the root and two products, and half a step 2^-149 where the product is subnormal
        check_scales(scales[0], most[None], 6 * ULP)
