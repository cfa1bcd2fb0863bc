"""route against a plain implementation: choices and the plan exactly, weights in 64 bits.

Tolerance of the weights: exp is off by at most 2 steps and its argument's difference by half a step of itself, a sum
over at most 512 experts takes 8 + 6 additions, then one division: (32 + |x - peak|) * 2^-24 relative."""
import pytest
import torch

import xgen_amd  # noqa: F401
from xgen_amd.operator.experts import route

pytestmark = pytest.mark.gpu


def reference(logits, k, bias=None, scoring="softmax", renormalize=True, first=0, local=None):
    x = logits.float().cpu()
    T, E = x.shape
    local = E - first if local is None else local
    score = x if bias is None else x + bias.cpu()
    score = torch.where(torch.isnan(score), torch.full_like(score, float("-inf")), score) + 0.0
    top, order = torch.sort(score, dim=1, descending=True, stable=True)
    taken = top[:, :k] > float("-inf")
    experts = torch.where(taken, order[:, :k], -1)
    xd = x.double()
    chosen = torch.where(taken, xd.gather(1, order[:, :k]), -torch.inf)
    if scoring == "sigmoid":
        w = torch.sigmoid(chosen)
        total = w.sum(1, keepdim=True) if renormalize else torch.ones(T, 1, dtype=torch.float64)
    else:
        peak = xd.amax(1, keepdim=True).clamp(min=-1e300)
        w = torch.exp(chosen - peak)
        total = (w if renormalize else torch.exp(xd - peak)).sum(1, keepdim=True)
    w = torch.where(taken, w / total, torch.zeros_like(w))
    w = torch.where(taken & torch.isnan(x).any(1, keepdim=True), torch.full_like(w, float("nan")), w)
    group = torch.where(taken & (experts >= first) & (experts < first + local), experts - first, local).reshape(-1)
    place = torch.argsort(group, stable=True)
    ends = torch.bincount(group, minlength=local + 1)[:local].cumsum(0)
    n = int(ends[-1])
    rows = torch.full((T * k,), -1)
    rows[:n] = place[:n] // k
    slots = torch.full((T * k,), -1)
    slots[place[:n]] = torch.arange(n)
    return w, experts, ends, rows, slots.reshape(T, k)


def check(cuda, logits, k, **kw):
    got = route(logits, k, **kw)
    names = dict(first="first_expert", local="local_experts")
    ref = reference(logits, k, **{{v: s for s, v in names.items()}.get(a, a): b for a, b in kw.items()})
    for name, g, r in zip(("experts", "ends", "rows", "slots"), got[1:], ref[1:]):
        assert g.dtype == torch.int32 and torch.equal(g.cpu().long(), r), name
    w, r = got.weights.cpu().double(), ref[0]
    assert torch.equal(torch.isnan(w), torch.isnan(r))
    spread = logits.float().cpu().double()
    spread = torch.where(torch.isfinite(spread), spread, torch.zeros_like(spread))
    tol = (32 + (spread.amax(1) - spread.amin(1)).abs().clamp(min=0))[:, None] * 2.0 ** -24
    ok = torch.isnan(r) | ((w - r).abs() <= tol * r + 2.0 ** -149)
    assert ok.all(), (w - r)[~ok]
    return got


def logits(cuda, T, E, seed, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return (torch.randn((T, E), generator=g, device=cuda) * scale).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("E,k", [(1, 1), (3, 3), (8, 2), (9, 4), (16, 16), (17, 1), (33, 5), (64, 6), (65, 8), (128, 8),
                                 (200, 32), (256, 7), (257, 3), (512, 32)])
def test_experts_and_choices(cuda, E, k, dtype):
    """bf16 logits repeat: ties go to the lowest expert."""
    for T in (5, 131, 333):
        check(cuda, logits(cuda, T, E, E + k + T, dtype), k)


@pytest.mark.parametrize("T", [1, 2, 8, 9, 16, 17, 32, 33, 63, 64, 65, 128, 129, 1000, 4096, 4097, 15624])
def test_token_counts(cuda, T):
    check(cuda, logits(cuda, T, 64, T), 6, renormalize=False)
    check(cuda, logits(cuda, T, 8, T, torch.bfloat16), 2)
    check(cuda, logits(cuda, T, 200, T), 5)


def test_chunks_of_several_pieces(cuda):
    """More tokens than one piece per workgroup covers, with a ragged last chunk."""
    check(cuda, logits(cuda, 32769 + 77, 16, 1), 2)
    check(cuda, logits(cuda, 100003, 8, 2, torch.bfloat16), 3, renormalize=False)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("scale", [1.0, 30.0])
def test_scoring_and_bias(cuda, scoring, renormalize, scale):
    x = logits(cuda, 300, 96, 3, scale=scale)
    bias = logits(cuda, 1, 96, 4)[0]
    check(cuda, x, 8, scoring=scoring, renormalize=renormalize)
    check(cuda, x, 8, bias=bias, scoring=scoring, renormalize=renormalize)


def test_masked_experts_and_rows(cuda):
    inf = float("inf")
    x = logits(cuda, 200, 24, 5)
    x[3] = -inf                   # a padding row: no expert
    x[4, 2:] = -inf               # two experts left for four choices
    x[5] = 0.0                    # all tied
    x[6, ::2], x[6, 1::2] = 0.0, -0.0
    x[7] = torch.finfo(torch.float32).min
    x[8, :20] = torch.finfo(torch.float32).min
    x[9, 5] = float("nan")
    x[10] = float("nan")
    x[199] = -inf
    for renormalize in (False, True):
        got = check(cuda, x, 4, renormalize=renormalize)
        assert (got.experts[[3, 199]] == -1).all() and not got.weights[[3, 199]].any()
        assert got.experts[4].tolist()[2:] == [-1, -1] and got.experts[5].tolist() == [0, 1, 2, 3]
        assert got.experts[6].tolist() == [0, 1, 2, 3]
        assert torch.isnan(got.weights[9]).all() and 5 not in got.experts[9].tolist()
        assert (got.experts[10] == -1).all() and not got.weights[10].any()
    x[11, 7] = inf
    assert route(x, 4).experts[11, 0] == 7 and torch.isnan(route(x, 4).weights[11, 0])
    everything = torch.full((70, 24), -inf, device=cuda)
    got = check(cuda, everything, 2)
    assert not got.ends.any() and (got.rows == -1).all()


@pytest.mark.parametrize("T", [40, 700])
def test_a_rank_s_experts(cuda, T):
    x = logits(cuda, T, 60, 6)
    whole = check(cuda, x, 6)
    for first, local in ((0, 20), (20, 20), (40, 20), (59, 1)):
        got = check(cuda, x, 6, first_expert=first, local_experts=local)
        assert torch.equal(got.experts, whole.experts) and torch.equal(got.weights, whole.weights)


def test_popular_expert(cuda):
    """All pairs of the first choice in one expert."""
    x = logits(cuda, 3000, 32, 7)
    x[:, 31] = 100.0
    got = check(cuda, x, 2)
    assert int(got.ends[31] - got.ends[30]) == 3000


def test_strides_and_no_tokens(cuda):
    x = logits(cuda, 90, 128, 8)
    check(cuda, x[:, 32:96], 4)
    check(cuda, x[::3, :64], 4)
    check(cuda, x.t()[:64], 4)
    check(cuda, x[:1].expand(70, 128), 4)
    got = route(x[:0], 4)
    assert [tuple(t.shape) for t in got] == [(0, 4), (0, 4), (128,), (0,), (0, 4)] and not got.ends.any()


def test_same_plan_on_every_run(cuda):
    x = logits(cuda, 5000, 128, 9, torch.bfloat16)
    first = route(x, 8)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, route(x, 8)))
