"""Products whose rows lie far apart, as one position of each of several sequences: the bits of contiguous rows."""
import pytest
import torch

import xgen_amd  # noqa: F401
from xgen_amd.operator.mxfp4 import mxfp4_matmul, quantize_mxfp4
from xgen_amd.ops import xops

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


def given(cuda, b, n, k, far):
    """rows, weights, a residual of [b, far / n, n]'s last positions, gates and indices."""
    g = torch.Generator(device=cuda).manual_seed(b)
    x, w = (torch.randn((r, k), generator=g, device=cuda).to(BF) for r in (b, n))
    stream = torch.zeros((b, far // n, n), dtype=BF, device=cuda)
    stream[:, -1] = torch.randn((b, n), generator=g, device=cuda).to(BF)
    table = torch.zeros((2, 1 << 27), dtype=BF, device=cuda)
    table[:, :n] = torch.randn((2, n), generator=g, device=cuda).to(BF)
    return x, w, stream[:, -1], table


@pytest.mark.parametrize("b", [1, 2, 5])
@pytest.mark.parametrize("far", [5376 * 1001, 5376 * 300])
def test_gated_residual_of_last_positions(cuda, b, far):
    n, k = 5376, 256
    x, w, res, table = given(cuda, b, n, k, far)
    idx = torch.zeros(b, dtype=torch.int64, device=cuda)
    gate = table[:1, :n]  # (one row: its stride says nothing)
    a, p = quantize_mxfp4(x), quantize_mxfp4(w)
    want = mxfp4_matmul(*a, *p, residual=res.clone(), gate_table=gate.clone(), indices=idx)
    assert torch.equal(mxfp4_matmul(*a, *p, residual=res, gate_table=gate, indices=idx), want)
    for dtype in (torch.int8, torch.float8_e4m3fn):
        (qa, sa), (qw, sw) = xops.quantize_rows(x, dtype), xops.quantize_rows(w, dtype)
        want = xops.scaled_mm_gate_residual(qa, qw, sa, sw, None, res.clone(), gate.clone(), idx)
        assert torch.equal(xops.scaled_mm_gate_residual(qa, qw, sa, sw, None, res, gate, idx), want)


@pytest.mark.parametrize("b", [1, 3, 300])
def test_packed_rows_far_apart(cuda, b):
    n, k, far = 96, 320, 9 << 20
    x, w, _, _ = given(cuda, b, n, k, n)
    a, p = quantize_mxfp4(x), quantize_mxfp4(w)
    wide = torch.zeros((b, far), dtype=torch.uint8, device=cuda)
    wide[:, :k // 2] = a[0]
    assert torch.equal(mxfp4_matmul(wide[:, :k // 2], a[1], *p), mxfp4_matmul(*a, *p))
    q, s = xops.quantize_rows(x, torch.int8)
    (qw, sw), wide = xops.quantize_rows(w, torch.int8), wide.view(torch.int8)
    wide[:, :k] = q
    got, want = (xops.scaled_mm(t, qw, s, sw, None, BF, 0, False)[0] for t in (wide[:, :k], q))
    assert torch.equal(got, want)
