"""Definitions in 64 bits for the tests of the operators with 8-bit operands, and what their outputs may be off by."""
import torch

DEV = "cuda:0"
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}
ULP = 2.0 ** -24                                    # half a step of fp32, relative


def matrix(rows, cols, dtype, extra=0, shift=0, device=DEV):
    """An empty matrix whose rows are `extra` elements further apart than they are long, `shift` elements into its memory; and the memory."""
    memory = torch.empty((rows * (cols + extra) + shift + 16), dtype=dtype, device=device)
    return memory[shift:shift + rows * (cols + extra)].view(rows, cols + extra)[:, :cols], memory


def widen(v, block_rows, blocks_shape):
    """One value per block -> one per element."""
    return v.repeat_interleave(block_rows, 0)[:blocks_shape[0]].repeat_interleave(128, 1)[:, :blocks_shape[1]]


def block_scales(v, block_rows):
    """max(largest magnitude / 448, 2^-126) of each block of a 64-bit matrix, [row blocks, column blocks]."""
    rows, cols = v.shape
    v = torch.nn.functional.pad(v, (0, -cols % 128, 0, -rows % block_rows))
    v = v.reshape(v.shape[0] // block_rows, block_rows, v.shape[1] // 128, 128)
    return (v.abs().amax((1, 3)) / 448).clamp_min(2.0 ** -126)


def check_8_bits(q, scales, v, block_rows, off):
    """q, scales against the 64-bit v, whose own values the kernel may have `off` (relative) away.  Scales [row blocks, column blocks]."""
    want = block_scales(v, block_rows)
    # the quotient by 448 is rounded once
    assert bool(((scales.double() - want).abs() <= want * (off + 2 * ULP)).all())
    # Numbers are within half a step of value / scale: 2^-4 of the power of two below it, 2^-10 where that is under 2^-6.  value / scale is off by
    # the value's own error, its scale's, and three roundings (scale, its inverse, the product).
    ratio = v / widen(want, block_rows, v.shape)
    half = torch.exp2(torch.floor(torch.log2(ratio.abs().clamp_min(2.0 ** -6)))) * 2.0 ** -4
    room = half + ratio.abs() * (2 * off + 8 * ULP)
    d = (q.double() - ratio).abs()
    assert bool((d <= room).all()), float((d / room).max())


def quantized(v, block_rows, rows_on=16):
    """(q with rows on 16-byte boundaries, scales as the product takes them) of an fp32 matrix: operands for tests, made with torch alone."""
    scales = block_scales(v.double(), block_rows).float()
    q, _ = matrix(v.shape[0], v.shape[1], TYPES["e4m3"], extra=-v.shape[1] % rows_on, device=v.device)
    q.copy_((v / widen(scales, block_rows, v.shape)).to(TYPES["e4m3"]))
    return q, (scales.t().contiguous() if block_rows == 1 else scales)


def round_room(want, dtype):
    """What the last rounding to the type may move a value by."""
    small = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}[dtype]
    return want.abs() * (torch.finfo(dtype).eps / 2) + small
