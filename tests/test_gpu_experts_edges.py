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


def aside(t, elements):
    """t's values in a contiguous view `elements` into its storage."""
    out = torch.empty(t.numel() + elements, dtype=t.dtype, device=t.device)[elements:].view(t.shape)
    return out.copy_(t)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("elements", [1, 2, 3])
def test_bias_at_an_odd_offset(cuda, dtype, elements):
    """A contiguous bias whose base is not on 16 bytes (one of 16-bit values not on 4 either): the same bits."""
    g = torch.Generator(device=cuda).manual_seed(elements)
    q, w = torch.randint(-99, 99, (90, 64), generator=g, device=cuda), torch.randint(-99, 99, (3, 208, 64), generator=g, device=cuda)
    s, ws = torch.rand((90,), generator=g, device=cuda), torch.rand((3, 208), generator=g, device=cuda) * 1e-3
    ends = torch.tensor([7, 7, 90], dtype=torch.int32, device=cuda)
    bias = torch.randn((3, 208), generator=g, device=cuda).to(dtype)
    call = (q.to(torch.int8), s, w.to(torch.int8), ws, ends)
    odd = aside(bias, elements)
    assert odd.is_contiguous() and odd.data_ptr() % 16 and torch.equal(odd, bias)
    assert torch.equal(grouped_matmul(*call, bias=odd), grouped_matmul(*call, bias=bias))
