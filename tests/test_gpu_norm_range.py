"""Root-mean-square norm of rows of finite values whose squares, or their sum, are beyond fp32: the result is of order 1 all the same."""
import pytest
import torch

from block8_util import DEV, TYPES, ULP, check_8_bits, round_room

pytestmark = pytest.mark.gpu

# As in test_gpu_norm_quantize.py (53 roundings up to 32768 columns); the factor 1 / rms is subnormal where the rms is above 2^126: half a step 2^-149
# beside 2^-128 is 2^-22, four halves of a unit.
OFF = 57 * ULP


def wanted(x, r, w, eps):
    h = (x + r).double() if r is not None else x.double()       # h is fp32; sums here are small beside the rounding that follows, or exact
    big = h.abs().amax(1, keepdim=True).clamp_min(1e-300)
    mean = (h / big).square().mean(1, keepdim=True)
    return h, h / big / torch.sqrt(mean + eps / big / big) * w.double()


def rows_of(rows, cols, kind, seed):
    """Ordinary rows, and among them rows of values from 1e17 up to the type's largest, of equal values, and with a single large one."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, cols, device=DEV, generator=g).clamp(-5, 5)
    for i, size in enumerate((3e17, 1e19, 1.9e19, 1e25, 1e31, 6e37)):
        x[i + 1::13] *= size
    x[7::13] = 3e38
    x[8::13, cols // 2] = -3.3e38
    w = 1 + 0.3 * torch.randn(cols, device=DEV, generator=g)
    return x.to(TYPES[kind]), w.to(TYPES[kind])


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("out", ["fp32", "bf16", "e4m3"])
@pytest.mark.parametrize("rows,cols", [(13, 1), (40, 96), (700, 4096), (40, 5001), (13, 9000), (13, 20480), (13, 20483), (26, 32768)])
def test_large_values(kind, out, rows, cols):
    from dlprimitives_b200 import capi
    x, w = rows_of(rows, cols, kind, cols)
    _, v = wanted(x, None, w, 1e-6)
    y = torch.empty(rows, cols, dtype=TYPES[out], device=DEV)
    scales = torch.empty(-(-cols // 128), rows, device=DEV) if out == "e4m3" else None
    capi.rms_norm(x, w, y, scales=scales)
    if out == "e4m3":
        check_8_bits(y, scales.t(), v, 1, OFF)
    else:
        # (small values beside one that is far larger end in subnormals of the output)
        assert bool(((y.double() - v).abs() <= round_room(v, y.dtype) + v.abs() * OFF + 2.0 ** -133).all())


@pytest.mark.parametrize("cols", [40000, 40001, 65537])
@pytest.mark.parametrize("place", ["total", "x"])
def test_long_rows_with_residual(cols, place):
    """Longer than a block's registers, with the total in a place of its own or in x's."""
    from dlprimitives_b200 import capi
    x, w = rows_of(13, cols, "fp32", cols)
    r = x / 8                                        # fp32 sums of these are rounded once, as the kernel's
    r[7::13] = 0
    r[8::13] = 0
    h, v = wanted(x, r, w, 1e-6)
    total = x if place == "x" else torch.empty_like(x)
    y = torch.empty_like(x)
    capi.rms_norm(x, w, y, residual=r, total=total)
    assert bool((total.double() == h).all())
    assert bool(((y.double() - v).abs() <= v.abs() * (2 * OFF) + 2.0 ** -133).all())


def test_eps_beside_large_squares():
    """The largest eps there is counts beside a mean of squares whose sum is just beyond fp32."""
    from dlprimitives_b200 import capi
    cols = 32768
    x = torch.full((2, cols), 1.5e17, device=DEV)    # sum of squares 7.4e38, mean 2.3e34
    w = torch.ones(cols, device=DEV)
    y = torch.empty_like(x)
    capi.rms_norm(x, w, y, eps=9.9e29)
    _, v = wanted(x, None, w, float(torch.tensor(9.9e29)))
    assert bool(((y.double() - v).abs() <= v.abs() * OFF).all())
    assert bool((1 - v > 1e-5).all())                # (eps is worth more than the room)


def test_what_is_not_finite_is_as_it_was():
    from dlprimitives_b200 import capi
    for cols in (384, 387, 40000):
        x = torch.full((4, cols), 1e30, device=DEV)
        x[1, 3] = float("inf")
        x[2, 3] = float("nan")
        y = torch.empty_like(x)
        capi.rms_norm(x, torch.ones(cols, device=DEV), y)
        assert bool(y[1, 3].isnan()) and bool((y[1, :3] == 0).all()) and bool((y[1, 4:] == 0).all())
        assert bool(y[2].isnan().all())
        assert bool(((y[[0, 3]] - 1).abs() <= OFF * 2).all())
