"""residual_norm against its formula in 64 bits, at the widths, strides, norms and row counts where it can go wrong.

Tolerances: every output is rounded once, by at most half a step (finfo.eps / 2 relative: bf16 2^-8, e4m3 2^-4; int8
half a unit of the row's scale).  In front of that the kernel computes in fp32: its chains have fewer than
64 roundings (at most 16 values per lane and accumulator, 10 steps of a reduction, and the products), so an
intermediate is off by at most C = 64 * 2^-24 of the magnitudes that enter it.  A norm divides by a deviation that
such errors enter too, so its result is off by C (1 + |n|) (1 + max|v| / deviation)."""
import pytest
import torch

import xgen_amd  # noqa: F401
from xgen_amd.operator.residual_norm import residual_norm

pytestmark = pytest.mark.gpu
C = 64 * 2.0 ** -24
FP8 = torch.float8_e4m3fn


def normed(v, kind, eps):
    """(normed v, 1 / deviation [.., 1])"""
    if kind is None:
        return v, torch.ones_like(v[..., :1])
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    r = 1 / (c.square().mean(-1, keepdim=True) + eps).sqrt()
    return c * r, r


def reference(x, y, *, branch_weight=None, gate_table=None, residual_scale=1.0, weight=None, scale=None, shift=None,
              indices=None, branch_norm="rms", norm="rms", eps=1e-6, **_):
    """(stream, rows, bound of the fp32 errors of each) in 64 bits."""
    one = torch.ones((), dtype=torch.float64, device=x.device)
    x, y = x.double(), y.double()
    wb = one if branch_weight is None else branch_weight.double()
    gate = one if gate_table is None else gate_table.double()[indices]
    n, r = normed(y, branch_norm, eps)
    branch = n * wb * gate
    err_b = (y.abs() if branch_norm is None else (1 + n.abs()) * (1 + y.abs().amax(-1, keepdim=True) * r)) * (wb * gate).abs()
    stream = residual_scale * x + branch
    err_s = (residual_scale * x).abs() + err_b
    h, r = normed(stream, norm, eps)
    w = one if weight is None else weight.double()
    sc = 0 * one if scale is None else scale.double()[indices]
    sh = 0 * one if shift is None else shift.double()[indices]
    rows = h * w * (1 + sc) + sh
    err_h = (1 + h.abs()) * (1 + err_s.amax(-1, keepdim=True) * r) * w.abs() * (1 + sc.abs()) + sh.abs()
    return stream, rows, C * err_s, C * err_h


def check(cuda, x, y, out_dtype=torch.bfloat16, **kw):
    got = residual_norm(x, y, out_dtype=out_dtype, **kw)
    stream, rows, err_s, err_h = reference(x, y, **kw)
    assert got[0].shape == x.shape and got[0].dtype == torch.bfloat16 and got[0].is_contiguous()
    half = 2.0 ** -8
    assert ((got[0].double() - stream).abs() <= half * stream.abs() + err_s * (1 + half)).all()
    if out_dtype == torch.bfloat16:
        assert got[1].shape == x.shape
        assert ((got[1].double() - rows).abs() <= half * rows.abs() + err_h * (1 + half)).all()
        return got
    rows, err_h = rows.flatten(0, 1), err_h.flatten(0, 1)
    q, s = got[1].double(), got[2].double()
    assert q.shape == rows.shape and s.shape == (rows.shape[0],)
    limit = 448.0 if out_dtype == FP8 else 127.0
    top = rows.abs().amax(1)
    assert ((s - top / limit).abs() <= (err_h.amax(1) + 8 * 2.0 ** -24 * top) / limit).all()
    # e4m3: half a step of the value, 2^-10 of the scale below the normal range; int8: half a unit
    step = 2.0 ** -4 * rows.abs() + 2.0 ** -10 * s[:, None] if out_dtype == FP8 else 0.5 * (1 + 2.0 ** -16) * s[:, None]
    assert ((q * s[:, None] - rows).abs() <= step + err_h * (1 + 2.0 ** -4) + 4 * 2.0 ** -24 * rows.abs()).all()
    assert (q.abs() <= limit).all() and (q.abs().amax(1) == limit).all()  # the row's largest value fills the format
    return got


def inputs(cuda, B, S, H, seed, offset=0.0, scale=3.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.randn((B, S, H), generator=g, device=cuda).bfloat16()
    y = (torch.randn((B, S, H), generator=g, device=cuda) * scale + offset).bfloat16()
    w = (1 + 0.1 * torch.randn((2, H), generator=g, device=cuda)).bfloat16()
    tables = (torch.randn((7, 3 * H), generator=g, device=cuda) * 0.3).bfloat16().chunk(3, dim=-1)
    idx = torch.randint(7, (S,), generator=g, device=cuda)
    return x, y, dict(branch_weight=w[0], weight=w[1], gate_table=tables[0], scale=tables[1], shift=tables[2], indices=idx)


@pytest.mark.parametrize("out", [torch.bfloat16, FP8, torch.int8])
@pytest.mark.parametrize("H", [8, 64, 504, 512, 520, 1024, 1032, 2040, 2056, 4096, 5376, 6152, 8192])
def test_widths(cuda, H, out):
    x, y, kw = inputs(cuda, 2, 9, H, seed=H)
    check(cuda, x, y, out, residual_scale=0.75, **kw)


@pytest.mark.parametrize("branch_norm", [None, "rms", "layer"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("H", [512, 2048])
def test_norms_and_what_is_left_out(cuda, norm, branch_norm, H):
    x, y, kw = inputs(cuda, 1, 33, H, seed=1)
    if branch_norm is None:
        kw.pop("branch_weight")
    check(cuda, x, y, branch_norm=branch_norm, norm=norm, **kw)
    for drop in (("gate_table",), ("scale", "shift"), ("weight",), ("gate_table", "scale", "shift", "indices")):
        check(cuda, x, y, branch_norm=branch_norm, norm=norm, **{k: v for k, v in kw.items() if k not in drop})
    check(cuda, x, y, FP8, branch_norm=branch_norm, norm=norm)


@pytest.mark.parametrize("offset", [30.0, 1000.0])
def test_layer_norm_of_rows_far_from_zero(cuda, offset):
    """Two-pass statistics: the variance of rows whose mean is far above their deviation."""
    x, y, kw = inputs(cuda, 1, 17, 2048, seed=2, offset=offset)
    check(cuda, x, y, branch_norm="layer", norm="layer", **kw)
    check(cuda, y, x, branch_norm="layer", norm="layer", **kw)


def test_f32_and_mixed_weights(cuda):
    x, y, kw = inputs(cuda, 1, 5, 1096, seed=3)
    check(cuda, x, y, **{**kw, "weight": kw["weight"].float() * 1.001, "branch_weight": kw["branch_weight"].float() * 0.999})
    check(cuda, x, y, **{**kw, "weight": kw["weight"].float() * 1.001})
    check(cuda, x, y, FP8, branch_weight=kw["branch_weight"].float())


def test_strided_views_and_unaligned_bases(cuda):
    x, y, kw = inputs(cuda, 3, 10, 1024, seed=4)
    wide = torch.cat([x, y], dim=-1)
    check(cuda, wide[..., :1024], wide[..., 1024:], **kw)                    # row stride 2,048
    check(cuda, x.transpose(0, 1).contiguous().transpose(0, 1), y, **kw)     # [S, B, H] in memory
    check(cuda, x[1:, ::2], y[1:, ::2], **{**kw, "indices": kw["indices"][::2]})  # strided indices, too
    check(cuda, x[:1].expand(3, 10, 1024), y, **kw)                          # one row block for every batch
    off = torch.empty(3 * 10 * 1024 + 4, dtype=torch.bfloat16, device=cuda)[4:].view(3, 10, 1024)  # 8 bytes off
    off.copy_(x)
    check(cuda, off, y, **kw)
    check(cuda, x[..., 8:1016], y[..., 8:1016], branch_norm="layer")         # rows start 16 bytes in
    check(cuda, x[..., 3:1003], y[..., 3:1003])                              # rows that 16-byte pieces cannot read


def test_one_row_and_no_rows(cuda):
    x, y, kw = inputs(cuda, 1, 1, 2048, seed=5)
    check(cuda, x, y, FP8, **kw)
    for shape in ((0, 3, 64), (2, 0, 64)):
        e = torch.empty(shape, dtype=torch.bfloat16, device=cuda)
        for out in (torch.bfloat16, FP8):
            got = residual_norm(e, e, out_dtype=out)
            assert got[0].shape == shape and got[1].numel() == 0


@pytest.mark.parametrize("H", [128, 5376])
def test_rows_do_not_touch_each_other(cuda, H):
    """NaN, infinities, zeros, a row of the type's largest values and an index outside the tables stay in their
    rows: the others' bits are those of a call without them."""
    x, y, kw = inputs(cuda, 1, 40, H, seed=6)
    clean = residual_norm(x, y, out_dtype=FP8, **kw)
    x2, y2, idx = x.clone(), y.clone(), kw["indices"].clone()
    x2[0, 3, 5], y2[0, 7, 1], y2[0, 11] = float("nan"), float("inf"), 0.0
    x2[0, 12], y2[0, 12] = 0.0, 0.0
    x2[0, 15] = torch.finfo(torch.bfloat16).max
    idx[20], idx[21], idx[39] = 7, -1, 1 << 40
    got = residual_norm(x2, y2, out_dtype=FP8, **{**kw, "indices": idx})
    touched = [3, 7, 11, 12, 15, 20, 21, 39]
    keep = torch.ones(40, dtype=torch.bool, device=cuda)
    keep[touched] = False
    assert torch.equal(clean[0][0, keep].view(torch.int16), got[0][0, keep].view(torch.int16))
    assert torch.equal(clean[1][keep].view(torch.uint8), got[1][keep].view(torch.uint8))
    assert torch.equal(clean[2][keep].view(torch.int32), got[2][keep].view(torch.int32))
    for r in (3, 7, 20, 21, 39):
        assert torch.isnan(got[2][r]) and torch.isnan(got[1][r].float()).all()
    for r in (20, 21, 39):
        assert torch.isnan(got[0][0, r].float()).all()
    assert torch.isfinite(got[2][[11, 12]]).all()
    # without a gate a bad index leaves the stream alone
    kw.pop("gate_table")
    got = residual_norm(x, y, **{**kw, "indices": idx})
    assert torch.isfinite(got[0].float()).all() and torch.isnan(got[1][0, 20].float()).all()


def test_zero_rows_quantize_to_zero(cuda):
    z = torch.zeros((1, 4, 256), dtype=torch.bfloat16, device=cuda)
    for out in (FP8, torch.int8):
        stream, q, s = residual_norm(z, z, out_dtype=out)
        assert not stream.float().any() and not q.float().any() and torch.isfinite(s).all()


def test_many_rows_of_a_long_sequence(cuda):
    """More rows than the grid holds at once, in two batches; the last ones too."""
    x, y, kw = inputs(cuda, 2, 20011, 264, seed=7)
    check(cuda, x, y, FP8, **kw)


@pytest.mark.parametrize("out", [torch.bfloat16, FP8])
def test_a_call_past_the_last_level_cache(cuda, out):
    x, y, kw = inputs(cuda, 1, 8000, 5376, seed=9)
    check(cuda, x, y, out, **kw)


def test_rows_past_32_bit_offsets(cuda):
    """x of 4.3 GB: rows whose byte offsets pass 2^32."""
    H, S = 8192, 262160
    x = torch.empty((1, S, H), dtype=torch.bfloat16, device=cuda)
    x[:, -300:] = torch.randn((1, 300, H), generator=torch.Generator(device=cuda).manual_seed(8), device=cuda).bfloat16()
    x[:, :-300] = 1.0
    got = residual_norm(x, x, norm="layer")
    stream, rows, err_s, err_h = reference(x[:, -300:], x[:, -300:], norm="layer")
    assert ((got[0][:, -300:].double() - stream).abs() <= 2.0 ** -8 * stream.abs() + 2 * err_s).all()
    assert ((got[1][:, -300:].double() - rows).abs() <= 2.0 ** -8 * rows.abs() + 2 * err_h).all()
    stream, rows, err_s, err_h = reference(x[:, :9], x[:, :9], norm="layer")
    assert ((got[1][:, :9].double() - rows).abs() <= 2.0 ** -8 * rows.abs() + 2 * err_h).all()
