"""What the draw's whole numbers leave out: masses are rounded to units of 2^-bits of the largest one, bits = min(51, 63 - ceil(log2(classes))), so a sum of
them is off by up to half a unit for each class, and a class of less than half a unit is never drawn.  One class with nearly all the mass and very many
equal ones around that limit, held to it."""
import math

import pytest
import torch

from block8_util import DEV

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [4000, 150001, 1 << 18, 1 << 22])
@pytest.mark.parametrize("place", ["first", "middle", "last"])
@pytest.mark.parametrize("share", [0.25, 0.499, 0.501, 0.75, 1.499, 1.501, 40.3])
def test_a_tail_of_masses_around_a_unit(n, place, share):
    from dlprimitives_b200 import capi
    bits = min(51, 63 - math.ceil(math.log2(n)))
    unit = 2.0 ** -bits
    high = {"first": 0, "middle": n // 2, "last": n - 1}[place]
    x = torch.full((1, n), math.log(share * unit), device=DEV)
    x[0, high] = 0.0
    w = float(torch.exp(x[0, 1 if high != 1 else 2].double()))                 # of one of the tail's classes, as it is in fp32
    before_high, whole = high * w, 1 + (n - 1) * w
    off = n * unit / 2 + unit                        # of a running sum, and of u times the whole one
    us = [0.0, 1e-9, 1e-7, 0.25, 0.5, 0.75, 1 - 2.0 ** -20, 1 - 2.0 ** -24]
    u = torch.tensor(us, device=DEV)
    tokens = torch.empty(len(us), dtype=torch.int32, device=DEV)
    capi.sample(x.expand(len(us), n).contiguous(), u, tokens)
    for v, t in zip(u.double().tolist(), tokens.tolist()):
        assert 0 <= t < n
        run = (t + 1) * w if t < high else before_high + 1 + (t - high) * w
        mass = 1.0 if t == high else w
        assert mass >= unit / 2 * (1 - 1e-6), (v, t)
        assert run > v * whole - 2 * off and run - mass <= v * whole + 2 * off, (v, t)
        if abs(v * whole - before_high) > 2 * off and abs(v * whole - before_high - 1) > 2 * off:
            assert (t == high) == (before_high <= v * whole < before_high + 1), (v, t)
