"""As many rows as a call can name."""
import pytest
import torch

from block8_util import DEV, TYPES

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [2 ** 31 - 8, 2 ** 31 - 7, 2 ** 31 - 1])
def test_quantize_rows_up_to_the_last_count(rows):
    from dlprimitives_b200 import capi
    x = torch.full((rows, 1), 2.0, dtype=torch.bfloat16, device=DEV)
    x[-1] = -7.0
    x[0] = 0.0
    q, scales = torch.zeros(rows, 1, dtype=torch.uint8, device=DEV).view(TYPES["e4m3"]), torch.zeros(1, rows, device=DEV)
    capi.quantize(x, q, scales)
    for at, value in ((0, 0.0), (1, 2.0), (rows // 2, 2.0), (rows - 9, 2.0), (rows - 2, 2.0), (rows - 1, -7.0)):
        assert float(q[at, 0].float()) == (448.0 if value > 0 else -448.0 if value < 0 else 0.0)
        assert float(scales[0, at]) == max(float(torch.tensor(abs(value)) / torch.tensor(448.0)), 2.0 ** -126)
