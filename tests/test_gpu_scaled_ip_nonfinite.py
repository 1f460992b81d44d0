"""What the activations of the product of 8-bit operands make of sums that are not finite, in each of its kernels: as everywhere in this library relu and
relu6 turn a NaN into 0, and the bounded ones give their bounds for an infinity."""
import math

import pytest
import torch

from block8_util import DEV, TYPES, quantized

pytestmark = pytest.mark.gpu

ACT = {"relu": lambda v: torch.where(v.isnan(), torch.zeros_like(v), v.clamp_min(0)), "relu6": lambda v: torch.where(v.isnan(), torch.zeros_like(v), v.clamp(0, 6)),
       "sigmoid": torch.sigmoid, "tanh": torch.tanh}


@pytest.mark.parametrize("kernel,rows,inputs,outputs", [("scaled_few", 7, 512, 300), ("scaled_few", 50, 512, 300), ("scaled_pair", 400, 512, 20000),
                                                        ("scaled_pair", 1000, 4096, 8000)])
@pytest.mark.parametrize("out", ["fp32", "bf16"])
def test_activations(kernel, rows, inputs, outputs, out):
    from dlprimitives_b200 import capi
    g = torch.Generator(device=DEV).manual_seed(rows)
    x, xs = quantized(torch.randn(rows, inputs, device=DEV, generator=g), 1)
    w, ws = quantized(torch.randn(outputs, inputs, device=DEV, generator=g) * inputs ** -0.5, 128)
    xs[1, 2] = math.nan
    xs[0, 3] = math.inf
    x.view(torch.uint8)[4, inputs - 1] = 0x7f        # NaN
    y = {}
    for act in ("identity", *ACT):
        y[act] = torch.empty(rows, outputs, dtype=TYPES[out], device=DEV)
        capi.scaled_inner_product(x, xs, w, ws, y[act], activation=act)
        assert capi.last_route()[0] == kernel
    plain = y["identity"].float()
    # before an activation what is computed from a value that is not finite is not finite either, and nothing else is touched
    assert bool(plain[2].isnan().all()) and bool(plain[4].isnan().all()) and not bool(plain[3].isfinite().any())
    assert bool((plain[3] == math.inf).any()) and bool((plain[3] == -math.inf).any())
    good = torch.ones(rows, dtype=torch.bool, device=DEV)
    good[2:5] = False
    assert bool(plain[good].isfinite().all())
    for act, f in ACT.items():
        got, want = y[act].float()[2:5], f(plain[2:5])
        assert bool(((got == want) | (got.isnan() & want.isnan())).all()), act
        assert bool(y[act][good].isfinite().all())
