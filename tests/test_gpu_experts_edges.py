"""Calls of route, grouped_matmul, combine and residual_norm at the edges of what they accept: no rows to take, views at
odd offsets, one token's view, scores and sizes at the ends of their ranges."""
import pytest
import torch

import xgen_amd  # noqa: F401
from test_experts_cpu import norm, outcome
from test_experts_edges_cpu import EPS_REFUSED, EPS_TAKEN
from test_gpu_route import reference
from xgen_amd.operator.experts import W8A8Experts, combine, grouped_matmul, route
from xgen_amd.operator.residual_norm import residual_norm

pytestmark = pytest.mark.gpu
xops = torch.ops.xgen_amd
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


# (the lowest and the highest logit of a token's row)
LOW = [(-95.0, -90.0), (-104.0, -88.0), (-200.0, -150.0), (-3e4, -2.9e4), (-100.0, -60.0), (-80.0, -1.0), (-1.0, 0.5), (-120.0, 40.0)]


def check_sigmoid(x, k, bias, renormalize):
    """The plan is test_gpu_route's; the weights in 64 bits by the sigmoids' logarithms, which do not underflow.

    Tolerance: as there (a sigmoid of a negative number is an exponential, a sum and a division, the sum below it one of k);
    a subnormal result is rounded by half of 2^-149."""
    got = route(x, k, bias=bias, scoring="sigmoid", renormalize=renormalize)
    ref = reference(x, k, bias=bias, scoring="sigmoid", renormalize=renormalize)
    for g, r in zip(got[1:], ref[1:]):
        assert torch.equal(g.cpu().long(), r)
    xd = x.double().cpu()
    log = torch.nn.functional.logsigmoid(xd).gather(1, ref[1].clamp(min=0))
    w = torch.softmax(log, 1) if renormalize else log.exp()
    tol = (32 + xd.amax(1) - xd.amin(1))[:, None] * 2.0 ** -24
    bad = (got.weights.cpu().double() - w).abs() > tol * w + 2.0 ** -149
    assert not bad.any(), (xd[bad.any(1)], got.weights.cpu()[bad], w[bad])
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("E,k", [(4, 3), (60, 8), (300, 32)])
@pytest.mark.parametrize("T", [len(LOW), 40 * len(LOW)])
def test_sigmoid_scores_of_low_logits(cuda, T, E, k, dtype):
    """Tokens whose sigmoids are subnormal or below every float: their quotients are not."""
    g = torch.Generator(device=cuda).manual_seed(E + T)
    lo, hi = torch.tensor(LOW * (T // len(LOW)), device=cuda).t()
    x = (lo[:, None] + (hi - lo)[:, None] * torch.rand((T, E), generator=g, device=cuda)).to(dtype)
    for bias in (None, torch.randn((E,), generator=g, device=cuda)):
        got = check_sigmoid(x, k, bias, True)
        assert ((got.weights.double().sum(1) - 1).abs() <= 40 * 2.0 ** -24).all()
        check_sigmoid(x, k, bias, False)


def test_sigmoid_scores_of_infinities(cuda):
    """-inf takes no part, +inf scores 1, a token of -inf alone takes nothing."""
    inf = float("inf")
    x = torch.tensor([[-inf, -300.0, -inf, -301.0], [inf, -100.0, -inf, 0.0], [-inf] * 4], device=cuda)
    for renormalize in (False, True):
        got = route(x, 3, scoring="sigmoid", renormalize=renormalize)
        assert got.experts.tolist() == [[1, 3, -1], [0, 3, 1], [-1] * 3] and not got.weights[2].any() and got.weights[0, 2] == 0
        total = 1.5 if renormalize else 1.0
        assert (got.weights[1, :2].double() - torch.tensor([1 / total, 0.5 / total], dtype=torch.float64, device=cuda)).abs().max() <= 2.0 ** -23
    assert (got.weights[0, :2].double() - torch.sigmoid(torch.tensor([1.0, -1.0], dtype=torch.float64, device=cuda))).abs().max() <= 8 * 2.0 ** -24


def one_row(t):
    """t [1, n] as a router's [n, 1] product transposed: strides (1, 1)."""
    v = torch.empty((t.shape[1], 1), dtype=t.dtype, device=t.device).t().copy_(t)
    assert v.shape == t.shape and v.stride() == (1, 1)
    return v


@pytest.mark.parametrize("E", [2, 24, 64, 200])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_token_whose_row_stride_is_short(cuda, E, dtype):
    """The stride between rows says nothing where there is one row."""
    g = torch.Generator(device=cuda).manual_seed(E)
    x = torch.randn((1, E), generator=g, device=cuda).to(dtype)
    for a, b in zip(route(one_row(x), 2), route(x, 2)):
        assert torch.equal(a, b)
    wide = torch.randn((7, E), generator=g, device=cuda).to(dtype)
    for a, b in zip(route(wide.as_strided((1, E), (0, 1)), 2), route(wide[:1], 2)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [torch.int8, FP8])
@pytest.mark.parametrize("activation", [0, 1])
def test_quantized_row_whose_stride_is_short(cuda, dtype, activation):
    g = torch.Generator(device=cuda).manual_seed(1)
    for H in (8, 50, 2048, 5376):
        x = torch.randn((1, H), generator=g, device=cuda).bfloat16()
        got, ref = xops.quantize_rows(one_row(x), dtype, activation), xops.quantize_rows(x, dtype, activation)
        assert torch.equal(got[0].view(torch.uint8), ref[0].view(torch.uint8)) and torch.equal(got[1], ref[1])


def test_experts_of_one_token_whose_stride_is_short(cuda):
    g = torch.Generator(device=cuda).manual_seed(2)
    up, down = (torch.randn(s, generator=g, device=cuda).bfloat16() for s in ((4, 64, 48), (4, 48, 32)))
    m = W8A8Experts(up, down, 2)
    x, logits = torch.randn((1, 48), generator=g, device=cuda).bfloat16(), torch.randn((1, 4), generator=g, device=cuda)
    ref = m(x, logits)
    assert ref.any() and torch.equal(m(one_row(x), one_row(logits)), ref)
    r = torch.randn((1, 48), generator=g, device=cuda).bfloat16()
    assert torch.equal(m(x, logits, residual=one_row(r)), m(x, logits, residual=r))
    y = torch.randn((1, 48), generator=g, device=cuda).bfloat16()
    w, s = torch.ones((1, 1), device=cuda), torch.zeros((1, 1), dtype=torch.int32, device=cuda)
    assert torch.equal(combine(one_row(y), w, s), y)


@pytest.mark.parametrize("eps", EPS_TAKEN + EPS_REFUSED)
def test_eps(cuda, eps):
    assert outcome(norm(eps=eps), cuda) == outcome(norm(eps=eps), "meta")
    z = torch.zeros((1, 3, 64), dtype=torch.bfloat16, device=cuda)
    if eps in EPS_TAKEN:  # rows of zeros stay zeros
        for kind in ("rms", "layer"):
            assert not any(t.any() for t in residual_norm(z, z, norm=kind, branch_norm=kind, eps=eps))


@pytest.mark.parametrize("scoring", [torch.sigmoid, lambda x: torch.softmax(x, 1)])
def test_a_bias_on_the_scores(cuda, scoring):
    """A router that ranks score + b: its biased scores as logits, its weights from the scores by the plan's experts.  By
    logits + b the order would be another one: expert 0 has the largest bias, and a score of almost nothing."""
    T, E, k, H = 300, 16, 4, 64
    g = torch.Generator(device=cuda).manual_seed(3)
    x = torch.rand((T, E), generator=g, device=cuda) * 0.2 - 0.1
    x[:, 0] = -40.0
    x[7] = float("-inf")
    b = torch.arange(E, 0, -1, device=cuda) / 4.0
    score = scoring(x).masked_fill(x == float("-inf"), 0.0)
    plan = route((score + b).masked_fill(x == float("-inf"), float("-inf")), k)
    w = score.gather(1, plan.experts.long().clamp(min=0)).masked_fill(plan.experts < 0, 0)
    w = w / w.sum(1, keepdim=True).clamp(min=torch.finfo(w.dtype).tiny)
    live = torch.arange(T, device=cuda) != 7
    top, order = torch.sort(scoring(x.double()) + b.double(), dim=1, descending=True)
    assert (top[live, :k] - top[live, 1:k + 1]).min() >= 2.0 ** -20  # plain in fp32, which is off by 2^-22 at most
    assert torch.equal(plan.experts[live].long(), order[live, :k]) and (plan.experts[live] == 0).any()
    assert (plan.experts[7] == -1).all()
    assert 0 not in route(x, k, bias=b, scoring="sigmoid").experts[live]
    y = torch.randn((T * k, H), generator=g, device=cuda).bfloat16()
    out = combine(y, w, plan.slots)
    s = scoring(x.double()).gather(1, order[:, :k])
    s = s / s.sum(1, keepdim=True)
    parts = y.double()[plan.slots.long().clamp(min=0)] * s[..., None]
    ref, mag = parts.sum(1)[live], parts.abs().sum(1)[live]
    # a score is off by 8 * 2^-24 (an exponential, a sum of 16, a division), a weight by two of them and 4 more roundings
    assert ((out[live].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (20 + k + 3) * 2.0 ** -24 * mag * 1.01).all()
    assert not out[7].any()
