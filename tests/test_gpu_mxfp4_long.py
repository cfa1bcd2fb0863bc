"""The 4-bit operators past 32-bit sizes: the same bits as calls of their rows alone."""
import pytest
import torch

import xgen_amd  # noqa: F401
from xgen_amd.operator.mxfp4 import dequantize_mxfp4, mxfp4_matmul, pack_scales, quantize_mxfp4

pytestmark = pytest.mark.gpu
BF, U8 = torch.bfloat16, torch.uint8


@pytest.mark.parametrize("m,seq", [(66051, 66051), (131200, 65600), (66054, 11009)])
def test_gated_sequences_past_one_launch(cuda, m, seq):
    """An output above 2 GiB in chunks of rows whose borders lie inside a sequence, one sequence and several."""
    n, k = 16384, 64
    g = torch.Generator(device=cuda).manual_seed(m)
    sa = torch.randint(120, 130, (m, k // 32), generator=g, device=cuda, dtype=U8)
    a = (torch.randint(0, 256, (m, k // 2), generator=g, device=cuda, dtype=U8), pack_scales(sa))
    w = (torch.randint(0, 256, (n, k // 2), generator=g, device=cuda, dtype=U8), pack_scales(torch.randint(120, 130, (n, k // 32), generator=g, device=cuda, dtype=U8)))
    res = torch.randn((m, n), generator=g, device=cuda, dtype=BF)
    gate = torch.randn((5, n), generator=g, device=cuda, dtype=BF)
    idx = torch.randint(0, 5, (seq,), generator=g, device=cuda)
    out = mxfp4_matmul(*a, *w, residual=res, gate_table=gate, indices=idx)
    for first in (0, 11009 - 100, 65024 - 300, 65280 - 300, 65600 - 300, m - 601, m - 1):
        last = min(m, first + 601)
        at = torch.arange(first, last, device=cuda) % seq
        part = mxfp4_matmul(a[0][first:last], pack_scales(sa[first:last]), *w, residual=res[first:last], gate_table=gate, indices=idx[at])
        assert torch.equal(out[first:last], part), first


def test_rows_past_one_launch(cuda):
    """More rows than a launch's threads: the last ones, and those at every launch's border, as calls of their own give them."""
    r, k, launch = (1 << 28) + 49, 32, 1 << 27
    base = torch.randn((1 << 20, k), generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).to(BF)
    x = torch.empty((r, k), dtype=BF, device=cuda)
    for first in range(0, r, len(base)):
        x[first:first + len(base)] = base[:r - first]
    codes, scales = quantize_mxfp4(x)
    back = dequantize_mxfp4(codes, scales)
    assert scales.shape == (1, r + 1, 8) and not scales[0, r].any()
    for first in (0, launch - 40, 2 * launch - 40, r - 49):
        last = min(r, first + 80)
        want = quantize_mxfp4(x[first:last])
        assert torch.equal(codes[first:last], want[0]) and torch.equal(scales[0, first:last], want[1][0, :last - first]), first
        assert torch.equal(back[first:last], dequantize_mxfp4(*want)), first
    period = codes[:len(base)]
    assert all(torch.equal(codes[f:f + len(base)], period[:r - f]) for f in range(0, r, 16 * len(base)))
