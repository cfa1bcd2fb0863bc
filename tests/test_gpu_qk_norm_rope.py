"""qk_norm_rope and rotary_table against plain implementations in 64 bits.

Tolerance of a rotated value out = s (d cw + d' sw), d = x - m: fp32 steps are 2^-24 of what they form.  s: the sum of
squares over at most 64 lanes of 8 values takes 8 + 6 additions, a multiplication, an addition and a reciprocal root
of one step: 12 (half of the sum's relative error, and the root's).  cw and sw one step each with the weight, the two
products, their sum and the scaling 4 more: 2^-24 * 20 * s (|d cw| + |d' sw|).  A mean of up to 14 additions moves d by
2^-24 * 16 * mean|x|, with another step of |x|: both partners', times s.  Then half a step of the output's type."""
import pytest
import torch

import xgen_amd  # noqa: F401
from xgen_amd.operator.qk_norm_rope import qk_norm_rope, rotary_frequencies, rotary_table

pytestmark = pytest.mark.gpu
BF, HF, F32, F64, I32, I64 = torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.int32, torch.int64


def reference(x, w, cos, sin, places, norm, eps, layout):
    """(values, tolerance before the last rounding) in 64 bits on the CPU."""
    x, half = x.double().cpu(), cos.shape[1]
    mean = x.mean(-1, keepdim=True) if norm == "layer" else torch.zeros_like(x[..., :1])
    d = x - mean
    s = torch.ones_like(mean) if norm is None else ((d * d).mean(-1, keepdim=True) + eps).rsqrt()
    w = torch.ones(x.shape[-1], dtype=F64) if w is None else w.double().cpu()
    v = d * w
    moved = ((16 * x.abs().mean(-1, keepdim=True) + x.abs() + mean.abs()) if norm == "layer" else torch.zeros_like(x)) * w.abs()
    if half:
        places = places.cpu()
        known = (places >= 0) & (places < len(cos))
        at = places.clamp(0, max(len(cos) - 1, 0))
        c, t = (torch.cat([a.double().cpu(), torch.zeros(1, half, dtype=F64)])[at].reshape(-1, x.shape[1], 1, half) for a in (cos, sin))
        i = slice(0, half) if layout == "half" else slice(0, 2 * half, 2)
        j = slice(half, 2 * half) if layout == "half" else slice(1, 2 * half, 2)
        out, size, shift = v.clone(), v.abs(), moved.clone()
        out[..., i], out[..., j] = v[..., i] * c - v[..., j] * t, v[..., j] * c + v[..., i] * t
        size[..., i] = (v[..., i] * c).abs() + (v[..., j] * t).abs()
        size[..., j] = (v[..., j] * c).abs() + (v[..., i] * t).abs()
        shift[..., i] = moved[..., i] + moved[..., j]
        shift[..., j] = shift[..., i]
        out = torch.where(known.reshape(-1, x.shape[1], 1, 1), out, torch.nan)
    return out * s, 2.0 ** -24 * s * (20 * size + shift)


def check(q, k, cos, sin, positions=None, q_weight=None, k_weight=None, norm="rms", eps=1e-6, layout="half"):
    got = qk_norm_rope(q, k, cos, sin, positions=positions, q_weight=q_weight, k_weight=k_weight, norm=norm, eps=eps, layout=layout)
    places = torch.arange(q.shape[1]) if positions is None else positions
    for x, w, y in ((q, q_weight, got[0]), (k, k_weight, got[1])):
        assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
        want, tol = reference(x, w, cos, sin, places, norm, eps, layout)
        y, info = y.double().cpu(), torch.finfo(x.dtype)
        assert torch.equal(torch.isnan(y), torch.isnan(want))
        off = torch.nan_to_num((y - want).abs() - tol - info.eps / 2 * (want.abs() + tol) - info.smallest_normal * info.eps, nan=0.0)
        assert bool((off <= 0).all()), float(off.max())
    return got


def angles(cuda, places, half, base=10000.0):
    f = rotary_frequencies(2 * half, base=base, device=cuda)[0]
    return rotary_table(torch.arange(places, device=cuda), f)


def heads(g, cuda, *shape, dtype=BF, scale=2.0, offset=0.0):
    return (torch.randn(shape, generator=g) * scale + offset).to(dtype).to(cuda)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("norm", ["rms", "layer", None])
@pytest.mark.parametrize("dim,half", [(128, 64), (128, 48), (64, 32), (64, 8), (256, 128), (512, 256), (32, 16), (16, 8), (8, 4), (96, 48), (80, 20),
                                      (72, 7), (40, 1), (264, 132), (120, 60)])
def test_heads(cuda, dim, half, norm, layout):
    g = torch.Generator().manual_seed(dim + half)
    cos, sin = angles(cuda, 11, half)
    w = [None if norm is None else 1 + 0.2 * torch.randn(dim, generator=g) for _ in range(2)]
    w = [t if t is None else t.to(BF).to(cuda) for t in w]
    check(heads(g, cuda, 2, 11, 5, dim), heads(g, cuda, 2, 11, 3, dim, offset=1.0), cos, sin, None, *w, norm=norm, layout=layout)


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("b,s,hq,hk", [(1, 1, 1, 1), (1, 1, 56, 56), (4, 1, 32, 8), (3, 17, 20, 4), (1, 501, 7, 1), (2, 3, 1, 0), (1, 5, 0, 3), (1, 2, 130, 130)])
def test_counts(cuda, b, s, hq, hk, dtype):
    g = torch.Generator().manual_seed(b + s + hq)
    cos, sin = angles(cuda, max(s, 4), 64)
    w = (1 + 0.1 * torch.randn(128, generator=g)).to(dtype).to(cuda)
    check(heads(g, cuda, b, s, hq, 128, dtype=dtype), heads(g, cuda, b, s, hk, 128, dtype=dtype), cos, sin, None, w, w)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_positions(cuda, layout):
    g = torch.Generator().manual_seed(1)
    cos, sin = angles(cuda, 131072, 48)
    q, k = heads(g, cuda, 3, 6, 4, 128), heads(g, cuda, 3, 6, 2, 128)
    own = torch.randint(0, 131072, (3, 6), generator=g)
    check(q, k, cos, sin, own.to(cuda), layout=layout)
    check(q, k, cos, sin, own[1].to(cuda), layout=layout)
    check(q, k, cos, sin, torch.stack([own[1], own[2]], 1).to(cuda)[:, 0], layout=layout)  # strided
    same = qk_norm_rope(q, k, cos, sin, positions=own[:1].expand(3, 6).to(cuda), layout=layout)
    for a, b in zip(same, qk_norm_rope(q, k, cos, sin, positions=own[0].to(cuda), layout=layout)):
        assert torch.equal(a, b)


def test_positions_outside(cuda):
    g = torch.Generator().manual_seed(2)
    cos, sin = angles(cuda, 9, 24)
    q, k = heads(g, cuda, 1, 6, 4, 64), heads(g, cuda, 1, 6, 1, 64)
    got = check(q, k, cos, sin, torch.tensor([0, 9, -1, 8, 1 << 40, -(1 << 63)], device=cuda))
    assert [bool(torch.isnan(got[0][0, i]).all()) for i in range(6)] == [False, True, True, False, True, True]
    check(q, k, cos[:3], sin[:3])                       # fewer places than tokens
    check(q, k, cos[:0], sin[:0])                       # none


def test_views(cuda):
    """Heads of a fused projection's rows, [B, H, S, D] transposed, every second token, bases and strides off 16 bytes, expanded."""
    g = torch.Generator().manual_seed(3)
    cos, sin = angles(cuda, 8, 32)
    fused = heads(g, cuda, 2, 8, 9 * 64)
    q, k = fused[..., :5 * 64].unflatten(-1, (5, 64)), fused[..., 5 * 64:7 * 64].unflatten(-1, (2, 64))
    want = check(q, k, cos, sin)
    for a, b in ((q.contiguous(), k.contiguous()), (q.transpose(1, 2).contiguous().transpose(1, 2), k)):
        for x, y in zip(qk_norm_rope(a, b, cos, sin), want):
            assert torch.equal(x, y)
    check(q[:, ::2], k[:, ::2], cos, sin)
    check(q[:1].expand(3, -1, -1, -1), k[1:].expand(3, -1, -1, -1), cos, sin)
    odd = heads(g, cuda, 2, 8, 5 * 64 + 3)[..., 3:].unflatten(-1, (5, 64))
    check(odd, k, cos, sin)
    table = torch.zeros((8, 70), device=cuda)
    table[:, 1:33], table[:, 35:67] = cos, sin
    for x, y in zip(qk_norm_rope(q, k, table[:, 1:33], table[:, 35:67]), want):
        assert torch.equal(x, y)
    flat = torch.zeros(2 * 8 * 32 + 1, device=cuda)     # contiguous tables off 16 bytes
    c, s = flat[1:257].view(8, 32).copy_(cos), flat[257:].view(8, 32).copy_(sin)
    for layout in ("half", "interleaved"):
        for x, y in zip(qk_norm_rope(q, k, c, s, layout=layout), qk_norm_rope(q, k, cos, sin, layout=layout)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("qt,kt", [(F32, F32), (BF, F32), (HF, HF), (None, BF), (F32, None), (BF, HF)])
def test_weights(cuda, qt, kt):
    g = torch.Generator().manual_seed(4)
    cos, sin = angles(cuda, 5, 64)
    w = [None if t is None else (1 + 0.2 * torch.randn(128, generator=g)).to(t).to(cuda) for t in (qt, kt)]
    check(heads(g, cuda, 1, 5, 6, 128), heads(g, cuda, 1, 5, 6, 128), cos, sin, None, *w)


def test_small_and_constant_heads(cuda):
    """Heads of zeros, of one value (no variance), of values whose squares leave fp32's normal range, and far from zero."""
    g = torch.Generator().manual_seed(5)
    cos, sin = angles(cuda, 4, 32)
    for norm in ("rms", "layer"):
        q = heads(g, cuda, 1, 4, 4, 64)
        q[0, 0], q[0, 1, 1], q[0, 2] = 0, 3.25, q[0, 2] * 2.0 ** -70
        check(q, q + 100, cos, sin, norm=norm)
        check(q, q, cos, sin, norm=norm, eps=1e-30)


def test_inf_in_one_pair_without_a_norm(cuda):
    """Without a norm nothing outside a pair sees its inf: the values past the rotated part and the other pairs stay."""
    g = torch.Generator().manual_seed(6)
    cos, sin = angles(cuda, 4, 16)
    q = heads(g, cuda, 1, 4, 2, 64)
    want = qk_norm_rope(q, q, cos, sin, norm=None)[0]
    q[0, 1, 0, 3] = float("inf")
    q[0, 2, 1, 50] = float("nan")
    got = qk_norm_rope(q, q, cos, sin, norm=None)[0]
    same = torch.ones((4, 2, 64), dtype=torch.bool)
    same[1, 0, 3] = same[1, 0, 19] = same[2, 1, 50] = False
    assert torch.equal(got[0].cpu()[same], want[0].cpu()[same]) and not torch.isfinite(got[0].cpu()[~same]).any()


def test_past_32_bit_offsets(cuda):
    """Rows whose offsets pass 2^32 bytes, read in place and written whole."""
    s, h = 150001, 130
    fused = torch.zeros((1, s, h, 128), dtype=BF, device=cuda)
    g = torch.Generator().manual_seed(7)
    at = [0, 1, 64528, 64529, 129055, 129056, s - 1]
    some = heads(g, cuda, 1, len(at), h, 128)
    fused[:, at] = some
    cos, sin = angles(cuda, s, 64)
    q, k = qk_norm_rope(fused[:, :, :100], fused[:, :, 100:], cos, sin)
    places = torch.tensor(at, device=cuda)
    a, b = qk_norm_rope(some[:, :, :100], some[:, :, 100:], cos, sin, positions=places)
    assert torch.equal(q[:, at], a) and torch.equal(k[:, at], b)
    assert int((q != 0).any(-1).sum()) == len(at) * 100


# ----------------------------------------------------------------------------- the table
def check_table(positions, f, axes=None, factor=1.0):
    """Half a step of fp32, the series' 2^-37, and the angle's own rounding to 64 bits (twice: here too)."""
    got = rotary_table(positions, f, axes=axes, factor=factor)
    p = positions.cpu().reshape(len(positions), -1)
    axis = torch.zeros(len(f), dtype=I64) if axes is None else axes.cpu().long()
    known = (axis >= 0) & (axis < p.shape[1])
    t = p[:, axis.clamp(0, p.shape[1] - 1)].double() * f.cpu()
    known = known & (t.abs() < 2.0 ** 36)
    for y, want in zip(got, (t.cos(), t.sin())):
        assert y.dtype == F32 and y.shape == t.shape
        y = y.double().cpu()
        assert torch.equal(torch.isnan(y), ~known)
        off = (y - factor * want).abs() - abs(factor) * (2.0 ** -24 * want.abs() + 2.0 ** -37 + t.abs() * 2.0 ** -52) - 1e-45
        assert bool((off[known] <= 0).all()), float(off[known].max())
    return got


@pytest.mark.parametrize("places,half", [(1, 1), (3, 64), (501, 48), (15624, 64), (7, 129)])
def test_table(cuda, places, half):
    g = torch.Generator().manual_seed(places)
    f = rotary_frequencies(2 * half, device=cuda)[0]
    check_table(torch.randint(0, 1000000, (places,), generator=g).to(cuda), f)


def test_table_axes(cuda):
    g = torch.Generator().manual_seed(8)
    f = torch.cat([rotary_frequencies(2 * n, device=cuda)[0] for n in (22, 21, 21)])
    axes = torch.tensor([0] * 22 + [1] * 21 + [2] * 21, dtype=I32, device=cuda)
    at = torch.randint(0, 128, (93, 3), generator=g).to(cuda)
    check_table(at, f, axes)
    check_table(at.t().contiguous().t(), f, axes)
    axes[5], axes[40] = 3, -1
    got = check_table(at, f, axes)
    assert torch.isnan(got[0][:, [5, 40]]).all()


def test_table_factor_and_far_positions(cuda):
    f = torch.tensor([1.0, 0.5, 1e-4, 31.0, 0.0, -2.0, float("inf"), float("nan")], dtype=F64, device=cuda)
    at = torch.tensor([0, 1, -1, -77, 2 ** 31, -(2 ** 31) - 5, 2 ** 35, 2 ** 37, 2 ** 62], device=cuda)
    check_table(at[:6], f[:6], factor=1.25)
    check_table(at, f[:6])
    got = rotary_table(at, f)
    assert torch.isnan(got[0][:, 6:]).all() and bool((got[0][:, 4] == 1).all()) and bool((got[1][:, 4] == 0).all())


def test_table_near_quarter_turns(cuda):
    """Angles at multiples of pi / 2 and beside them, where one of the two is next to nothing."""
    f = torch.tensor([torch.pi / 2, torch.pi / 4, torch.pi / 2 * (1 + 1e-9)], dtype=F64, device=cuda)
    check_table(torch.arange(-9, 10, device=cuda), f)
