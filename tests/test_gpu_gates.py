"""The gated activations where their factor is small: against a * logistic(2 z) * b in 64 bits, which loses nothing there, with a bound beside the value
itself (a result of 0, of the wrong sign or of another size fails)."""
import math

import pytest
import torch

from block8_util import DEV, TYPES, ULP, check_8_bits

pytestmark = pytest.mark.gpu


def argument(a, how):
    return a if how == "silu" else 2 * math.sqrt(2 / math.pi) * (a + 0.044715 * a ** 3)


def room(a, how):
    """Relative.  silu: 10 halves of a unit, as in test_gpu_norm_quantize.py.  gelu: its argument t = 1.5957.. (a + 0.0447.. a^3) has no cancellation; the cube's
    term has a constant and two roundings, the sum one, the product with 1.5957.. a constant and one: 6 halves, which e^-t passes on as 6 |t|, weighted
    with e^-t / (1 + e^-t) <= 1."""
    t = argument(a, how)
    return (10 + (6 * t.abs() * torch.sigmoid(-t) if how == "gelu" else 0)) * ULP


@pytest.mark.parametrize("kind", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("how", ["silu", "gelu"])
@pytest.mark.parametrize("cols", [8, 7])
def test_one_value_to_a_block(kind, how, cols):
    from dlprimitives_b200 import capi
    n = 1 << 17
    g = torch.Generator(device=DEV).manual_seed(cols)
    lo, hi = (-80.0, 20.0) if how == "silu" else (-9.0, 6.0)
    x = torch.zeros(n, 2 * cols, dtype=TYPES[kind], device=DEV)
    x[:, 3] = (lo + (hi - lo) * torch.rand(n, device=DEV, generator=g)).to(x.dtype)
    x[:, cols + 3] = (1 + torch.rand(n, device=DEV, generator=g)).to(x.dtype)
    q, scales = torch.empty(n, cols, dtype=TYPES["e4m3"], device=DEV), torch.empty(1, n, device=DEV)
    capi.quantize(x, q, scales, gate=how)
    a, b = x[:, 3].double(), x[:, cols + 3].double()
    want = a * torch.sigmoid(argument(a, how)) * b
    got = q[:, 3].double() * scales[0].double()
    # the number is 448 or -448, the scale the value / 448 rounded once; 2^-126 the lowest scale, and a step of it
    seen = want.abs() >= 448 * 2.0 ** -126
    assert int(seen.sum()) > n // 2
    off = (got - want).abs() / want.abs()
    assert bool((off <= room(a, how) + 2 * ULP)[seen].all()), float((off / room(a, how))[seen].max())
    assert bool(((got - want).abs() <= 2.0 ** -126 * 32)[~seen].all())         # half a step of the numbers up to 448, in units of the lowest scale


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(300, 1000), (37, 1001), (2, 12288)])
def test_gelu_of_negative_rows(kind, rows, cols):
    from dlprimitives_b200 import capi
    g = torch.Generator(device=DEV).manual_seed(rows)
    x = torch.randn(rows, 2 * cols, device=DEV, generator=g)
    x[:, :cols] = -1 - 5 * torch.rand(rows, cols, device=DEV, generator=g)
    x = x.to(TYPES[kind])
    q, scales = torch.empty(rows, cols, dtype=TYPES["e4m3"], device=DEV), torch.empty(-(-cols // 128), rows, device=DEV)
    capi.quantize(x, q, scales, gate="gelu")
    a, b = x[:, :cols].double(), x[:, cols:].double()
    off = float(room(torch.tensor([-6.03], dtype=torch.float64), "gelu"))      # bf16 rounds -5.99 to -6
    check_8_bits(q, scales.t(), a * torch.sigmoid(argument(a, "gelu")) * b, 1, off)
