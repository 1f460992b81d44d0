"""Root-mean-square norm and the 8-bit form of a matrix, against their definitions in 64 bits."""
import math

import pytest
import torch

from block8_util import DEV, TYPES, ULP, block_scales, check_8_bits, matrix, round_room

pytestmark = pytest.mark.gpu

# Sums of squares: a thread adds at most cols / 512 + 8 squares one after the other, then 5 steps over the lanes and 16 over the warps; the mean, the
# root and two products follow.  The root halves the sum's error.  Up to 32768 columns that is under (64 + 8 + 21) / 2 + 6 roundings.
OFF = 53 * ULP


def norm_case(rows, cols, kind, seed, extra=0, shift=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    t = TYPES[kind]
    x, r, total = (matrix(rows, cols, t, extra, shift)[0] for _ in range(3))
    x.copy_(torch.randn(rows, cols, device=DEV, generator=g))
    r.copy_(4 * torch.randn(rows, cols, device=DEV, generator=g))
    w = (1 + 0.3 * torch.randn(cols, device=DEV, generator=g)).to(t)
    return x, r, total, w


def norm_wanted(x, r, w, eps):
    h = x.double() + (r.double() if r is not None else 0)
    return h, h / torch.sqrt(h.square().mean(1, keepdim=True) + eps) * w.double()


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("out", ["fp32", "fp16", "bf16", "e4m3"])
@pytest.mark.parametrize("rows,cols,extra,shift", [(1, 1, 0, 0), (3, 127, 0, 0), (5, 128, 0, 0), (2, 136, 8, 8), (4, 1000, 24, 0), (3, 4096, 0, 0),
                                                  (2, 4097, 0, 0), (1, 16384, 0, 0), (2, 20001, 3, 1), (700, 96, 0, 0), (2, 32768, 0, 0)])
def test_norm(kind, out, rows, cols, extra, shift):
    from dlprimitives_b200 import capi
    x, r, total, w = norm_case(rows, cols, kind, rows + cols, extra, shift)
    y, memory = matrix(rows, cols, TYPES[out], extra, shift)
    memory.view(torch.uint8).fill_(0x5a)
    guard = memory.clone()
    scales = torch.full((-(-cols // 128), rows), -1.0, device=DEV) if out == "e4m3" else None
    capi.rms_norm(x, w, y, residual=r, total=total, scales=scales, eps=1e-5)
    h, v = norm_wanted(x, r, w, 1e-5)
    assert bool(((total.double() - h).abs() <= round_room(h, x.dtype) + h.abs() * ULP).all())
    if out == "e4m3":
        check_8_bits(y, scales.t(), v, 1, OFF)
    else:
        assert bool(((y.double() - v).abs() <= round_room(v, y.dtype) + v.abs() * OFF).all())
    # what lies between the rows and around them is as it was
    y.view(torch.uint8).fill_(0x5a)
    assert torch.equal(memory.view(torch.uint8), guard.view(torch.uint8))


@pytest.mark.parametrize("cols", [50000, 65537])
def test_norm_of_long_rows(cols):
    """Longer than what a block of threads holds at once."""
    from dlprimitives_b200 import capi
    x, r, total, w = norm_case(2, cols, "bf16", cols)
    y = torch.empty(2, cols, device=DEV)
    capi.rms_norm(x, w, y, residual=r, total=r, eps=1e-6)          # total in the residual's place
    _, r0, _, _ = norm_case(2, cols, "bf16", cols)
    h, v = norm_wanted(x, r0, w, 1e-6)
    assert bool(((y.double() - v).abs() <= v.abs() * (2 * OFF)).all())
    assert bool(((r.double() - h).abs() <= round_room(h, r.dtype) + h.abs() * ULP).all())


@pytest.mark.parametrize("cols", [512, 333])
@pytest.mark.parametrize("place", ["x", "residual"])
def test_norm_in_place(cols, place):
    from dlprimitives_b200 import capi
    x, r, total, w = norm_case(33, cols, "bf16", 5)
    y, y2 = torch.empty_like(x), torch.empty_like(x)
    capi.rms_norm(x, w, y, residual=r, total=total)
    capi.rms_norm(x, w, y2, residual=r, total=x if place == "x" else r)
    assert torch.equal(y, y2) and torch.equal(total, x if place == "x" else r)


def test_norm_without_residual_and_special_rows():
    from dlprimitives_b200 import capi
    x, _, _, w = norm_case(6, 384, "fp32", 9)
    x[1] = 0
    x[2, 130] = math.nan
    x[3, 5] = math.inf
    x[4] = 0
    x[4, 383] = 1e-30
    y = torch.empty(6, 384, dtype=TYPES["e4m3"], device=DEV)
    scales = torch.empty(3, 6, device=DEV)
    capi.rms_norm(x, w, y, scales=scales, eps=1e-6)
    z = torch.empty(6, 384, device=DEV)
    capi.rms_norm(x, w, z, eps=1e-6)
    _, v = norm_wanted(x, None, w, 1e-6)
    for rows in ([0, 1, 4, 5],):
        check_8_bits(y[rows], scales.t()[rows], v[rows], 1, OFF)
        assert bool(((z[rows].double() - v[rows]).abs() <= v[rows].abs() * OFF).all())
    assert bool((scales[:, 1] == 2.0 ** -126).all()) and bool((y[1].float() == 0).all())
    assert bool(z[2].isnan().all()) and bool(scales[:, 2].isnan().all())
    value = y.float() * scales.t().repeat_interleave(128, 1)
    assert bool(value[2].isnan().all())
    assert bool(value[3, 5].isnan()) and bool(z[3, 5].isnan())             # inf / inf; the rest of the row is finite / inf
    assert bool((z[3, :5] == 0).all())


def gate(a, b, kind):
    if kind == "silu":
        return a * torch.sigmoid(a) * b
    return 0.5 * a * (1 + torch.tanh(math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3))) * b


# silu: the exponential within 2^-22.5 (3 halves of a unit), its correction and the sum with 1 a half each, the reciprocal within a unit (2), two products:
# 9 halves; 10 with the constants.  gelu: its argument has four roundings and the constants', and e^-2z passes an argument's error d on as 2 |z| d,
# weighted with 1 - 1 / (1 + e^-2z) <= 1: for a >= -1, where 2 |z| (1 - ..) is under 1.3, another 6 halves.
GATE_OFF = {"none": 0.0, "silu": 10 * ULP, "gelu": 16 * ULP}


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("how", ["none", "silu", "gelu"])
@pytest.mark.parametrize("rows,cols,extra,shift", [(1, 1, 0, 0), (3, 127, 0, 0), (5, 128, 0, 0), (2, 136, 16, 16), (4, 1000, 1, 3), (3, 4096, 0, 0),
                                                  (1, 12289, 0, 0), (2000, 24, 0, 0)])
def test_quantize_rows(kind, how, rows, cols, extra, shift):
    from dlprimitives_b200 import capi
    g = torch.Generator(device=DEV).manual_seed(rows + cols)
    x, _ = matrix(rows, cols * (1 if how == "none" else 2), TYPES[kind], extra, shift)
    x.copy_(3 * torch.randn(x.shape, device=DEV, generator=g))
    if how == "gelu":
        x[:, :cols].clamp_(min=-1.0)               # further down 1 + tanh loses its leading bits, in fp32 as in any type: see the test below
    q, memory = matrix(rows, cols, TYPES["e4m3"], extra, shift)
    memory.view(torch.uint8).fill_(0x5a)
    guard = memory.clone()
    scales = torch.empty(-(-cols // 128), rows + 2, device=DEV)[:, :rows]
    capi.quantize(x, q, scales, gate=how)
    v = x.double() if how == "none" else gate(x[:, :cols].double(), x[:, cols:].double(), how)
    check_8_bits(q, scales.t(), v, 1, GATE_OFF[how])
    q.view(torch.uint8).fill_(0x5a)
    assert torch.equal(memory.view(torch.uint8), guard.view(torch.uint8))


@pytest.mark.parametrize("how", ["silu", "gelu"])
def test_gates_far_out(how):
    """Arguments where the exponential over- or underflows, and where gelu's 1 + tanh cancels: the error stays small beside the argument."""
    from dlprimitives_b200 import capi
    a = torch.tensor([-1e30, -300.0, -100.0, -89.0, -20.0, -6.0, -3.0, -1e-20, 0.0, 1e-20, 3.0, 20.0, 100.0, 300.0, 1e4, 1e12], device=DEV)
    x = torch.ones(16, 256, device=DEV)
    x[:, :128] = 0                                   # one value to a block: its number is 448 or 0, its scale the value / 448
    x[:, 0] = a
    q = torch.empty(16, 128, dtype=TYPES["e4m3"], device=DEV)
    scales = torch.empty(1, 16, device=DEV)
    capi.quantize(x, q, scales, gate=how)
    got = q[:, 0].double() * scales[0].double()
    want = gate(a.double(), torch.ones_like(a).double(), how)
    # 1 + tanh is off by at most four halves of a unit of 1, times half the argument; the 8 bits hold one value by its scale exactly but for roundings
    room = want.abs() * 20 * ULP + (a.double().abs().clamp_max(20) * 4 * ULP if how == "gelu" else 0) + 448 * 2.0 ** -126
    assert bool(((got - want).abs() <= room).all()), (got, want)


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows,cols,extra,shift", [(1, 1, 0, 0), (128, 128, 0, 0), (129, 130, 0, 0), (300, 1000, 8, 8), (127, 4099, 2, 1), (1000, 257, 0, 0)])
def test_quantize_weights(kind, rows, cols, extra, shift):
    from dlprimitives_b200 import capi
    g = torch.Generator(device=DEV).manual_seed(rows + cols)
    x, _ = matrix(rows, cols, TYPES[kind], extra, shift)
    x.copy_(0.05 * torch.randn(rows, cols, device=DEV, generator=g))
    q, memory = matrix(rows, cols, TYPES["e4m3"], extra, shift)
    memory.view(torch.uint8).fill_(0x5a)
    guard = memory.clone()
    scales = torch.empty(-(-rows // 128), -(-cols // 128), device=DEV)
    capi.quantize(x, q, scales, block_rows=128)
    check_8_bits(q, scales, x.double(), 128, 0.0)
    q.view(torch.uint8).fill_(0x5a)
    assert torch.equal(memory.view(torch.uint8), guard.view(torch.uint8))


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantize_of_very_many_rows(block_rows):
    # more blocks of 128 rows than a grid's second axis has; the last rows against the same rows by themselves
    from dlprimitives_b200 import capi
    rows, tail = 65536 * 128 + 130, 258
    x = torch.randn(rows, 8, device=DEV).to(torch.bfloat16)
    q, part = torch.empty(rows, 8, dtype=TYPES["e4m3"], device=DEV), torch.empty(tail, 8, dtype=TYPES["e4m3"], device=DEV)
    scales = torch.empty((1, rows) if block_rows == 1 else (-(-rows // 128), 1), device=DEV)
    part_scales = torch.empty((1, tail) if block_rows == 1 else (-(-tail // 128), 1), device=DEV)
    capi.quantize(x, q, scales, block_rows=block_rows)
    capi.quantize(x[-tail:], part, part_scales, block_rows=block_rows)
    assert torch.equal(q[-tail:].view(torch.uint8), part.view(torch.uint8))
    assert torch.equal(scales.flatten()[-part_scales.numel():], part_scales.flatten())


def test_quantize_blocks_that_are_not_finite_or_zero():
    from dlprimitives_b200 import capi
    x = torch.randn(260, 384, device=DEV)
    x[:128, :128] = 0
    x[130, 129] = math.nan
    x[257, 300] = -math.inf
    x[128:256, 256:] = 1e-42                        # subnormal
    for block_rows in (1, 128):
        q = torch.empty(260, 384, dtype=TYPES["e4m3"], device=DEV)
        shape = (3, 260) if block_rows == 1 else (3, 3)
        scales = torch.empty(shape, device=DEV)
        capi.quantize(x, q, scales, block_rows=block_rows)
        s = scales.t() if block_rows == 1 else scales
        assert bool((s[0, 0] == 2.0 ** -126).all()) and bool((q[:128, :128].float() == 0).all())
        at = (slice(130, 131), 257) if block_rows == 1 else (1, 2)
        assert bool(s[at[0], 1].isnan().all()) and bool(s[at[1], 2].isinf().all())
        value = q.double() * s.double().repeat_interleave(block_rows, 0)[:260].repeat_interleave(128, 1)
        assert bool(value[130, 128:256].isnan().all()) and bool(value[257, 300].isnan())
        fine = torch.ones(260, 384, dtype=torch.bool, device=DEV)
        if block_rows == 1:
            fine[130, 128:256] = fine[257, 256:] = False
        else:
            fine[128:256, 128:256] = fine[256:, 256:] = False
        want = block_scales(torch.where(fine, x, torch.zeros_like(x)).double(), block_rows)
        assert bool((value.isfinite() == fine).all())
        assert bool(((s.double() - want).abs() <= 2 * ULP * want)[s.isfinite() & (want > 2.0 ** -126)].all())
