"""mxfp4_matmul on each tile of its choice, with every epilogue and a bias, to one rounding.

Tolerance: ceil(K / 64) * 2^-22 * sum |a w| of the sums (tests/test_gpu_mxfp4.py), 2^-24 of the biased value for the bias's
addition; of GELU |gelu'| <= 1.13 times that and 2^-20 of |y| for its own arithmetic; of a gated residual |gate| times that and
2^-24 of the result; then half a step of the output's type, and no other."""
import pytest
import torch

import xgen_amd  # noqa: F401
from test_gpu_mxfp4 import gelu, packed, split, tile, values
from xgen_amd.operator.mxfp4 import mxfp4_matmul, pack_scales, unpack_scales

pytestmark = pytest.mark.gpu
BF, HF, F32, F64 = torch.bfloat16, torch.float16, torch.float32, torch.float64
TILES = [(32, 64), (32, 128), (64, 64), (64, 128), (128, 128), (128, 192), (256, 128), (256, 192), (256, 256)]


def smallest_shapes(gated):
    """The smallest ragged shape of one launch that runs on each tile."""
    found = {}
    for m in (1, 30, 61, 125, 251, 501, 1003, 1955, 3906, 7811):
        for n in (1040, 2064, 5392, 14352):
            for k in (96, 2080, 7136, 14304):
                t = tile(m, n, k, gated)
                if not split(m, n, k, gated) and (t not in found or m * n * k < found[t][0] * found[t][1] * found[t][2]):
                    found[t] = (m, n, k)
    return found


def sample(g, m):
    return torch.cat([torch.arange(min(m, 40)), torch.randperm(m, generator=g)[:60], torch.arange(max(0, m - 40), m)]).unique()


def taken(a, at, m, k):
    """Rows `at` of packed rows."""
    return a[0][at.cuda()], pack_scales(unpack_scales(a[1], m, k)[at.cuda()])


def check(got, a, w, m, n, k, bias=None, activation=None, res=None, t=None):
    """got [m, n] of rows a; t: each row's gate."""
    av, wv = values(a, m, k).cuda(), values(w, n, k).cuda()
    y = av @ wv.t().contiguous()
    error = -(-k // 64) * 2.0 ** -22 * (av.abs() @ wv.abs().t().contiguous())
    if bias is not None:
        y = y + bias.double()
        error = error + 2.0 ** -24 * (y.abs() + error)
    if activation:
        error, y = 1.13 * error + 2.0 ** -20 * y.abs() + 1e-30, gelu(y)
    if res is not None:
        y = res.double() + y * t.double()
        error = error * t.double().abs() + 2.0 ** -24 * y.abs()
    f = torch.finfo(got.dtype)
    error = error + f.eps / 2 * (y.abs() + error) + f.smallest_normal * f.eps
    off = (got.double() - y).abs() - error
    assert bool((off <= 0).all()), (float(off.max()), divmod(int(off.argmax()), n))


def given(g, m, n, t, seq, dtype=BF):
    """bias, residual, gate table and indices."""
    return (torch.randn(n, generator=g).to(dtype).cuda(), torch.randn((m, n), generator=g).to(BF).cuda(),
            torch.randn((t, n), generator=g).to(BF).cuda(), torch.randint(0, t, (seq,), generator=g).cuda())


@pytest.mark.parametrize("want", TILES)
@pytest.mark.parametrize("form", ["plain", "gelu", "gated"])
def test_tile(cuda, want, form):
    gated = form == "gated"
    shapes = smallest_shapes(gated)
    assert set(shapes) == set(TILES)
    m, n, k = shapes[want]
    print("tile", want, "of", (m, n, k), flush=True)
    g = torch.Generator().manual_seed(m + n)
    a, w = packed(g, m, k, spread=0), packed(g, n, k, 0.02, spread=0)
    bias, res, gate, idx = given(g, m, n, 7, m, F32)
    at = sample(g, m)
    rows, here = taken(a, at, m, k), at.to(cuda)
    kw = dict(residual=res, gate_table=gate, indices=idx) if gated else dict(activation="gelu_tanh", out_dtype=HF) if form == "gelu" else {}
    got = mxfp4_matmul(*a, *w, bias=bias, **kw)
    more = dict(res=res[here], t=gate[idx[here]]) if gated else dict(activation=True) if form == "gelu" else {}
    check(got[here], rows, w, len(at), n, k, bias, **more)
    # the same rows in a call of their own, on another tile: the same bits
    kw = dict(residual=res[here], gate_table=gate, indices=idx[here]) if gated else kw
    assert torch.equal(got[here], mxfp4_matmul(*rows, *w, bias=bias, **kw))


@pytest.mark.parametrize("batch,seq,n,k", [(1, 1, 16, 32), (1, 5, 96, 160), (3, 41, 272, 320), (7, 3, 1040, 2080), (2, 501, 1024, 1056), (5, 391, 2064, 608)])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_gated_residual_with_a_bias(cuda, batch, seq, n, k, dtype):
    """Odd sequences, every type of bias; views of the residual, the table and the bias give the same bits."""
    g = torch.Generator().manual_seed(seq + n)
    m = batch * seq
    a, w = packed(g, m, k, spread=0), packed(g, n, k, 0.05, spread=0)
    bias, res, gate, idx = given(g, m, n, 6, seq, dtype)
    got = mxfp4_matmul(a[0].reshape(batch, seq, -1), a[1], *w, bias=bias, residual=res.reshape(batch, seq, n), gate_table=gate, indices=idx)
    check(got.reshape(m, n), a, w, m, n, k, bias, res=res, t=gate[idx.repeat(batch)])
    for apart in (8, 3):  # rows apart, in place and copied
        wide = [torch.zeros((len(t), n + apart), dtype=BF, device=cuda) for t in (res, gate)]
        for t, into in zip((res, gate), wide):
            into[:, apart:] = t
        views = [t[:, apart:] for t in wide]
        off = torch.cat([bias[:1], bias])[1:]
        assert torch.equal(mxfp4_matmul(*a, *w, bias=off, residual=views[0], gate_table=views[1], indices=idx), got.reshape(m, n))


@pytest.mark.parametrize("m,n,k", [(1, 16, 32), (5, 96, 160), (200, 400, 768), (700, 2048, 512), (1955, 528, 320)])
@pytest.mark.parametrize("dtype,bias,activation", [(BF, BF, "gelu_tanh"), (HF, HF, "gelu_tanh"), (BF, F32, "gelu_tanh"), (HF, F32, None), (BF, HF, None)])
def test_epilogue(cuda, m, n, k, dtype, bias, activation):
    g = torch.Generator().manual_seed(m + k)
    a, w = packed(g, m, k, spread=0), packed(g, n, k, 0.05, spread=0)
    b = given(g, 1, n, 1, 1, bias)[0]
    check(mxfp4_matmul(*a, *w, bias=b, out_dtype=dtype, activation=activation), a, w, m, n, k, b, activation)
