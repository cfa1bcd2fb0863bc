"""quantize_rows on more rows than one launch's threads, at widths that a workgroup takes row by row."""
import pytest
import torch

import xgen_amd  # noqa: F401
from xgen_amd.ops import xops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", [torch.int8, torch.float8_e4m3fn])
def test_rows_past_one_launch(cuda, out):
    rows, cols, piece = (1 << 24) + 39, 3, 1 << 20
    x = torch.empty((rows, cols), dtype=torch.bfloat16, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(1)
    for first in range(0, rows, piece):
        last = min(rows, first + piece)
        x[first:last] = torch.randn((last - first, cols), generator=g, device=cuda).to(torch.bfloat16)
    q, scale = xops.quantize_rows(x, out)
    for first in range(0, rows, piece):
        last = min(rows, first + piece)
        want = xops.quantize_rows(x[first:last].clone(), out)
        assert torch.equal(q[first:last].view(torch.uint8), want[0].view(torch.uint8)) and torch.equal(scale[first:last], want[1]), first
