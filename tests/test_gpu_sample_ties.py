"""Draws where a prefix ends among logits of 16 bits that are far below zero, or around it, and equal by the hundred: which of them are kept goes by index."""
import pytest
import torch

from block8_util import DEV, TYPES
from test_gpu_sample import check, settings

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("which", ["p", "k", "kp", "tp", "tkpm"])
@pytest.mark.parametrize("n", [600, 866, 5003, 13906, 127517])
@pytest.mark.parametrize("middle,spread", [(-1000.0, 3.0), (-1000.0, 0.01), (-3.0, 0.05), (-0.02, 0.01), (1000.0, 3.0), (-60000.0, 100.0)])
def test_many_equal_logits(kind, which, n, middle, spread):
    g = torch.Generator(device=DEV).manual_seed(n)
    rows = 6
    x = (middle + spread * torch.randn(rows, n, device=DEV, generator=g)).to(TYPES[kind])
    if kind == "fp32":
        x = x.bfloat16().float()
    kw = settings(rows, n, which, g)
    if "top_k" in kw:                                # up to all of them
        kw["top_k"] = (1 + n * torch.rand(rows, device=DEV, generator=g)).int()
    if "temperature" in kw:                          # far up too, where all logits count
        kw["temperature"] *= torch.tensor([1.0, 1.0, 30.0, 1000.0, 0.1, 100.0], device=DEV)
    # u away from its ends: what the masses' rounding leaves out does not show
    check(x, 0.01 + 0.98 * torch.rand(rows, device=DEV, generator=g), kw)
