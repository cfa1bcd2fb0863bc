"""Calls of route, grouped_matmul, combine and residual_norm at the edges of what they accept: no rows to take, views at
odd offsets, one token's view, scores and sizes at the ends of their ranges."""
import pytest
import torch

import xgen_amd  # noqa: F401
from xgen_amd.operator.experts import grouped_matmul

pytestmark = pytest.mark.gpu
FP8 = torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [torch.int8, FP8])
@pytest.mark.parametrize("scales", [0, 1])
@pytest.mark.parametrize("M", [1, 40, 700])
def test_rows_of_an_activation_without_rows(cuda, dtype, scales, M):
    """Every index is outside an activation of no rows: NaN rows up to the last end, zeros behind it; neither the
    activation nor its scale (an empty tensor has no address) is read."""
    q = torch.empty((0, 64), dtype=torch.uint8, device=cuda).view(dtype)
    w = torch.zeros((3, 48, 64), dtype=torch.uint8, device=cuda).view(dtype)
    ends = torch.tensor([(M + 1) // 2, (M + 1) // 2, M - M // 4], dtype=torch.int32, device=cuda)
    rows = torch.arange(M, dtype=torch.int32, device=cuda) - 1
    for sw in (torch.ones(3, 48, device=cuda), torch.ones(3, device=cuda)):
        out = grouped_matmul(q, torch.ones(scales, device=cuda), w, sw, ends, rows=rows)
        last = int(ends[-1])
        assert torch.isnan(out[:last].float()).all() and not out[last:].any()
