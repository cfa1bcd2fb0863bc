"""The operators of a block with experts and sandwich norms that are timed, and what their outputs are compared with.

Four operators, in the order a block runs them: the norm behind the attention branch with the gated residual and the
norm in front of the feed-forward (`residual_norm`), the router with its plan of which rows go to which expert
(`route`), the experts' W8A8 products over ragged row groups (`grouped_matmul`), and the weighted sum of each token's
expert rows (`combine`).  Widths are d = 5,376 with its 14,336-wide feed-forward, tokens 15,624, 3,906, 1,955 and 501
as elsewhere in this package, and generic sizes of models with many small experts (2,048 wide, 64 or 128 experts).

Formulas, all in real numbers (outputs are rounded once, to their type):

  residual_norm  stream = a x + gate[i] * norm_b(y) * w_b;   h = norm(stream) * w * (1 + scale[i]) + shift[i]
                 norm: RMS  v / sqrt(mean(v^2) + eps)  or layer  (v - mean) / sqrt(var + eps); i = indices[position]
                 h as bf16, or as e4m3fn rows: s = max(max|h| / 448, FLT_MIN), q = e4m3fn(h / s)
  route          the k experts of largest logit + bias (float32 sum; ties to the lowest index, -inf never chosen);
                 weights softmax(logits) at them, divided by their sum if renormalised; rows sorted by (expert, token, choice)
  grouped_matmul out[m] = (q[rows[m]] . w[e]^T) * (a_scale[rows[m]] * w_scale[e]) + bias[e], m in group e
  combine        out[t] = residual[t] + gate[i] * sum_j weights[t, j] * y[slots[t, j]]
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
TABLE_ROWS = 20
FLT_MIN = 1.17549435082228750797e-38
EPS = 1e-6
MOST_WEIGHTS = 8 * 14336 * 5376          # elements of the largest listed case's experts
MOST_FLOPS = 2 * 15624 * 2 * 14336 * 5376


def listed():
    return [
        # one new token of two requests between two blocks of a model without modulation: the smallest call
        dict(name="norm_2", op="norm", batch=2, seq=1, d=2048, branch_norm="rms", norm="rms", gated=False, out="bf16"),
        # a small image request's block: gate and modulation tables, quantized for the following projection
        dict(name="norm_501_fp8", op="norm", batch=1, seq=501, d=5376, branch_norm="rms", norm="layer", gated=True, out="fp8"),
        # the same at a 5 s clip's token share, as the block without a quantized projection takes it
        dict(name="norm_15624", op="norm", batch=1, seq=15624, d=5376, branch_norm="rms", norm="rms", gated=True, out="bf16"),
        # a decoding step of four requests
        dict(name="route_4", op="route", tokens=4, experts=64, k=6, dtype="f32", padded=0, renormalize=True, biased=False),
        # a clip's token share with its padding rows, many experts, balanced by a bias
        dict(name="route_15624", op="route", tokens=15624, experts=128, k=8, dtype="bf16", padded=311, renormalize=True, biased=True),
        # a decoding step of eight requests: most experts get no row or one, their weights are what is read
        dict(name="grouped_8", op="grouped", kind="fp8", tokens=8, experts=64, k=6, kk=2048, n=2816, gather=True, bias=False, acc="mfma"),
        # a prompt through many small experts, up-projection reading each token's row for its experts
        dict(name="grouped_2049", op="grouped", kind="fp8", tokens=2049, experts=128, k=8, kk=2048, n=1536, gather=True, bias=False, acc="mfma"),
        # down-projection of a medium request in INT8
        dict(name="grouped_1955_int8", op="grouped", kind="int8", tokens=1955, experts=64, k=6, kk=1408, n=2048, gather=False, bias=False, acc="exact"),
        # a dual-stream block: text and video rows with weights of their own, products summed exactly
        dict(name="streams_4162", op="streams", kind="fp8", text=256, video=3906, kk=5376, n=5376, bias=True, acc="exact"),
        # the largest: two of eight wide experts per token at a 5 s clip's share
        dict(name="grouped_15624", op="grouped", kind="fp8", tokens=15624, experts=8, k=2, kk=5376, n=14336, gather=True, bias=True, acc="mfma"),
        # the decoding step's sum
        dict(name="combine_8", op="combine", tokens=8, experts=64, k=6, d=2048, padded=0, gated=False),
        # the clip's sum (its padding rows have no expert), with the gated residual behind it
        dict(name="combine_15624", op="combine", tokens=15624, experts=8, k=2, d=5376, padded=311, gated=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "route", "route", "grouped", "grouped", "grouped", "streams", "combine", "combine"])
    tokens = _log_int(rng, 1, 15624)
    experts = rng.choice([4, 8, 16, 60, 64, 128, 160, 256])
    k = rng.randint(1, min(8, experts))
    if op == "norm":
        batch = rng.choice([1, 1, 2, 3])
        return dict(op=op, batch=batch, seq=max(1, tokens // batch), d=8 * rng.randint(64, 672), branch_norm=rng.choice(["rms", "layer", "none"]),
                    norm=rng.choice(["rms", "layer"]), gated=rng.random() < 0.6, out=rng.choice(["bf16", "fp8"]))
    if op == "route":
        return dict(op=op, tokens=tokens, experts=experts, k=k, dtype=rng.choice(["bf16", "f32", "f16"]),
                    padded=rng.choice([0, 0, 1]) * (tokens // 7), renormalize=rng.random() < 0.5, biased=rng.random() < 0.5)
    if op == "combine":
        return dict(op=op, tokens=tokens, experts=experts, k=min(k, 4) if tokens > 8000 else k, d=8 * rng.randint(64, 672),
                    padded=rng.choice([0, 0, 1]) * (tokens // 7), gated=rng.random() < 0.5)
    kind = rng.choice(["fp8", "fp8", "int8"])
    acc = "exact" if kind == "int8" else rng.choice(["mfma", "mfma", "exact"])
    kk, n = 16 * rng.randint(32, 336), 16 * rng.randint(32, 336)
    if op == "streams":
        return dict(op=op, kind=kind, text=rng.randint(1, 512), video=_log_int(rng, 64, 8000), kk=kk, n=n, bias=rng.random() < 0.5, acc=acc)
    while experts * kk * n > MOST_WEIGHTS // 2:
        experts //= 2
    k = min(k, experts)
    while 2 * tokens * k * kk * n > MOST_FLOPS // 4:
        tokens = max(1, tokens // 2)
    return dict(op=op, kind=kind, tokens=tokens, experts=experts, k=k, kk=kk, n=n, gather=rng.random() < 0.6, bias=rng.random() < 0.4, acc=acc)


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _logits(g, tokens, experts, padded=0, dtype=torch.float32):
    """Router logits of popular and unpopular experts; the last `padded` tokens may go nowhere."""
    x = torch.randn((tokens, experts), generator=g, device=DEV) + 0.3 * torch.randn((experts,), generator=g, device=DEV)
    if padded:
        x[tokens - padded:] = float("-inf")
    return x.to(dtype)


def _plain_route(logits, bias, k, renormalize):
    """weights [T, k], experts [T, k], group ends [E], tokens [T k], slots [T, k]."""
    tokens, count = logits.shape
    x = logits.float()
    score = x if bias is None else x + bias
    top, chosen = torch.sort(score, dim=1, descending=True, stable=True)
    top, chosen = top[:, :k], chosen[:, :k]
    taken = top > float("-inf")
    peak = x.amax(dim=1, keepdim=True)
    p = torch.exp(x - torch.where(peak > float("-inf"), peak, torch.zeros_like(peak)))
    w = torch.where(taken, p.gather(1, chosen), torch.zeros_like(top))
    total = w.sum(dim=1, keepdim=True) if renormalize else p.sum(dim=1, keepdim=True)
    w = torch.where(taken, w / total, torch.zeros_like(w))
    group = torch.where(taken, chosen, count).reshape(-1)
    order = torch.argsort(group, stable=True)
    ends = torch.zeros(count + 1, dtype=torch.int64, device=x.device).scatter_add_(0, group, torch.ones_like(group)).cumsum(0)[:count]
    place = torch.arange(tokens * k, device=x.device)
    routed = place < ends[-1]
    rows = torch.where(routed, order // k, -1)
    slots = torch.zeros_like(place).scatter_(0, order, torch.where(routed, place, -1)).reshape(tokens, k)
    ids = torch.where(taken, chosen, -1)
    return w, ids.int(), ends.int(), rows.int(), slots.int()


def _quantized(g, shape, kind):
    """8-bit values as a symmetric quantization leaves them (a few at the limit)."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16 if math.prod(shape) > 1 << 24 else torch.float32)
    if kind == "int8":
        return x.mul_(32).round_().clamp_(-127, 127).to(torch.int8)
    return x.mul_(112).clamp_(-448, 448).to(torch.float8_e4m3fn)


def _scales(g, count, mean):
    return torch.exp(0.5 * torch.randn((count,), generator=g, device=DEV)) * mean


def _tables(g, d, count):
    """`count` column blocks of one table, as a block's modulation rows are kept."""
    return _randn(g, TABLE_ROWS, count * d, scale=0.1).chunk(count, dim=-1)


def _inputs(case, seed):
    g, op = _gen(seed), case["op"]
    if op == "norm":
        shape, d = (case["batch"], case["seq"], case["d"]), case["d"]
        given = dict(x=_randn(g, *shape), y=_randn(g, *shape, scale=3.0), w=1 + _randn(g, d, scale=0.1),
                     wb=None if case["branch_norm"] == "none" else 1 + _randn(g, d, scale=0.1), a=1.0, gate=None, scale=None, shift=None, indices=None)
        if case["gated"]:
            gate, scale, shift = _tables(g, d, 3)
            given.update(gate=gate, scale=scale, shift=shift, indices=torch.randint(0, TABLE_ROWS, (case["seq"],), generator=g, device=DEV), a=0.75)
        return given
    if op == "route":
        dtype = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[case["dtype"]]
        return dict(logits=_logits(g, case["tokens"], case["experts"], case["padded"], dtype),
                    bias=0.2 * torch.randn((case["experts"],), generator=g, device=DEV) if case["biased"] else None)
    if op == "combine":
        w, _, _, _, slots = _plain_route(_logits(g, case["tokens"], case["experts"], case["padded"]), None, case["k"], True)
        given = dict(y=_randn(g, case["tokens"] * case["k"], case["d"]), w=w, slots=slots, residual=None, gate=None, indices=None)
        if case["gated"]:
            given.update(residual=_randn(g, case["tokens"], case["d"]), gate=_tables(g, case["d"], 2)[1],
                         indices=torch.randint(0, TABLE_ROWS, (case["tokens"],), generator=g, device=DEV))
        return given
    kind, kk, n = case["kind"], case["kk"], case["n"]
    if op == "streams":
        ends = torch.tensor([case["text"], case["text"] + case["video"]], dtype=torch.int32, device=DEV)
        experts, count, rows = 2, case["text"] + case["video"], None
    else:
        experts = case["experts"]
        _, _, ends, tokens, _ = _plain_route(_logits(g, case["tokens"], experts), None, case["k"], True)
        rows = tokens if case["gather"] else None
        count = case["tokens"] if case["gather"] else case["tokens"] * case["k"]
    return dict(q=_quantized(g, (count, kk), kind), s=_scales(g, count, 0.01), w=_quantized(g, (experts, n, kk), kind),
                ws=_scales(g, experts * n, 0.0002).reshape(experts, n), ends=ends, rows=rows,
                bias=_randn(g, experts, n, scale=0.01) if case["bias"] else None)


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if case["op"] in ("grouped", "streams"):  # the largest group: what the plain form pads every group to
        ends = state["ends"].long()
        state["most"] = int((ends - torch.cat([ends.new_zeros(1), ends[:-1]])).max())
    return state


# ----------------------------------------------------------------------------- plain forms
def _norm(v, kind):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(dim=-1, keepdim=True)
    return v * torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + EPS)


def _plain_norm(s):
    case = s["case"]
    branch = _norm(s["y"].float(), case["branch_norm"])
    if s["wb"] is not None:
        branch = branch * s["wb"].float()
    if s["gate"] is not None:
        branch = branch * s["gate"].float()[s["indices"]]
    stream = s["a"] * s["x"].float() + branch
    h = _norm(stream, case["norm"]) * s["w"].float()
    if s["scale"] is not None:
        h = h * (1 + s["scale"].float()[s["indices"]]) + s["shift"].float()[s["indices"]]
    if case["out"] == "bf16":
        return stream.bfloat16(), h.bfloat16()
    h = h.reshape(-1, case["d"])
    scale = (h.abs().amax(dim=1) / 448.0).clamp(min=FLT_MIN)
    return stream.bfloat16(), (h / scale[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn), scale


def _plain_grouped(s):
    """Every group padded to the largest one, as one batched product."""
    q, ends, rows, most = s["q"], s["ends"].long(), s["rows"], s["most"]
    total = q.shape[0] if rows is None else rows.shape[0]
    at = (ends - torch.diff(ends, prepend=ends.new_zeros(1)))[:, None] + torch.arange(most, device=q.device)
    valid = at < ends[:, None]
    at = at.clamp(max=total - 1)
    source = at if rows is None else rows.long()[at].clamp(min=0)
    y = torch.bmm(q[source.reshape(-1)].float().reshape(*source.shape, -1), s["w"].float().transpose(1, 2))
    y = y * (s["s"][source][:, :, None] * s["ws"][:, None, :])
    if s["bias"] is not None:
        y = y + s["bias"].float()[:, None, :]
    out = torch.zeros((total, s["w"].shape[1]), dtype=torch.bfloat16, device=q.device)
    out[at[valid]] = y[valid].bfloat16()
    return out


def _plain_combine(s):
    taken = s["slots"] >= 0
    rows = s["y"][s["slots"].long().clamp(min=0)].float()
    out = torch.where(taken[:, :, None], rows * s["w"][:, :, None], torch.zeros((), device=rows.device)).sum(dim=1)
    if s["gate"] is not None:
        out = out * s["gate"].float()[s["indices"]]
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return out.bfloat16()


# ----------------------------------------------------------------------------- the framework's operators
_API = []


def _api():
    if not _API:
        from xgen_amd.operator.experts import combine, grouped_matmul, route
        from xgen_amd.operator.residual_norm import residual_norm
        _API.append((residual_norm, route, grouped_matmul, combine))
    return _API[0]


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        residual_norm, route, grouped_matmul, combine = _api()
        if op == "norm":
            return residual_norm(state["x"], state["y"], branch_weight=state["wb"], gate_table=state["gate"], residual_scale=state["a"],
                                 weight=state["w"], scale=state["scale"], shift=state["shift"], indices=state["indices"],
                                 branch_norm=None if case["branch_norm"] == "none" else case["branch_norm"], norm=case["norm"], eps=EPS,
                                 out_dtype=torch.bfloat16 if case["out"] == "bf16" else torch.float8_e4m3fn)
        if op == "route":
            return tuple(route(state["logits"], case["k"], bias=state["bias"], renormalize=case["renormalize"]))
        if op == "combine":
            return combine(state["y"], state["w"], state["slots"], residual=state["residual"], gate_table=state["gate"], indices=state["indices"])
        return grouped_matmul(state["q"], state["s"], state["w"], state["ws"], state["ends"], rows=state["rows"], bias=state["bias"],
                              accumulation=case["acc"])
    if op == "norm":
        return _plain_norm(state)
    if op == "route":
        return _plain_route(state["logits"], state["bias"], case["k"], case["renormalize"])
    if op == "combine":
        return _plain_combine(state)
    return _plain_grouped(state)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "norm":
        rows, d = case["batch"] * case["seq"], case["d"]
        tables = 3 * min(TABLE_ROWS, case["seq"]) if case["gated"] else 0
        out = 2 * d if case["out"] == "bf16" else d + 4
        return {"bytes": rows * (6 * d + out) + (2 + tables) * 2 * d, "flops": 16 * rows * d}
    tokens = case.get("tokens", 0)
    if op == "route":
        size = 4 if case["dtype"] == "f32" else 2
        return {"bytes": tokens * (case["experts"] * size + 16 * case["k"]) + 4 * case["experts"], "flops": 4 * tokens * case["experts"]}
    if op == "combine":
        d, rows = case["d"], tokens * case["k"]
        return {"bytes": 2 * d * (rows + tokens * (2 if case["gated"] else 1)) + 8 * rows, "flops": 2 * rows * d}
    kk, n = case["kk"], case["n"]
    if op == "streams":
        rows = read = case["text"] + case["video"]
        used = 2.0
    else:
        rows, experts = tokens * case["k"], case["experts"]
        read = tokens if case["gather"] else rows
        used = experts * (1 - (1 - case["k"] / experts) ** tokens)  # experts that get a row, of an even router
    return {"bytes": read * (kk + 4) + used * n * (kk + 4) + rows * 2 * n, "flops": 2 * rows * n * kk}


# ----------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op == "norm":
        def normed(v, kind):
            if kind == "none":
                return v
            c = v - v.sum(-1, keepdim=True) / v.shape[-1] if kind == "layer" else v
            return c / ((c ** 2).sum(-1, keepdim=True) / v.shape[-1] + EPS).sqrt()

        def row(table):
            return table.double().index_select(0, s["indices"])

        b = normed(s["y"].double(), case["branch_norm"])
        b = b if s["wb"] is None else b * s["wb"].double()
        b = b if s["gate"] is None else b * row(s["gate"])
        stream = s["x"].double() * s["a"] + b
        h = normed(stream, case["norm"]) * s["w"].double()
        if s["scale"] is not None:
            h = h + h * row(s["scale"]) + row(s["shift"])
        if case["out"] == "bf16":
            return stream, h
        h = h.flatten(0, 1)
        top = (h.abs().max(dim=1).values / 448).clamp(min=FLT_MIN)
        # the nearest e4m3fn value: a step of 2^(exponent - 3), 2^-9 at least
        v = h / top[:, None]
        step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
        return stream, (torch.round(v / step) * step).clamp(-448, 448), top
    if op == "route":
        x, count = s["logits"].double(), case["experts"]
        score = s["logits"].float() if s["bias"] is None else s["logits"].float() + s["bias"]
        # rank by counting: the experts ahead of each one
        tokens, k = x.shape[0], case["k"]
        index = torch.arange(count, device=x.device)
        w = torch.zeros((tokens, k), dtype=torch.float64, device=x.device)
        for at in range(0, tokens, 512):
            c = score[at:at + 512]
            ahead = (c[:, None, :] > c[:, :, None]) | ((c[:, None, :] == c[:, :, None]) & (index[None, None, :] < index[None, :, None]))
            rank = torch.where(c > float("-inf"), ahead.sum(2), count)
            e = torch.softmax(x[at:at + 512], dim=1).nan_to_num(0.0)
            for j in range(k):
                w[at:at + 512, j] = (e * (rank == j)).sum(1)
        if case["renormalize"]:
            total = w.sum(1, keepdim=True)
            w = torch.where(total > 0, w / total, w)
        return w, None, None, None, None
    if op == "combine":
        out = torch.zeros((case["tokens"], case["d"]), dtype=torch.float64, device=DEV)
        for j in range(case["k"]):
            there = s["slots"][:, j].long()
            out[there >= 0] += (s["w"][:, j:j + 1].double() * s["y"].index_select(0, there.clamp(min=0)).double())[there >= 0]
        if case["gated"]:
            out = s["residual"].double() + out * s["gate"].double().index_select(0, s["indices"])
        return out
    if 2 * case["kk"] * case["n"] * (case["tokens"] * case["k"] if op == "grouped" else case["text"] + case["video"]) > 2e13:
        return None
    source = torch.arange(s["q"].shape[0], device=DEV) if s["rows"] is None else s["rows"].long()
    out = torch.zeros((source.shape[0], case["n"]), dtype=torch.float64, device=DEV)
    begin = 0
    for e, end in enumerate(s["ends"].tolist()):
        if end > begin:
            a = s["q"].index_select(0, source[begin:end]) if case["kind"] == "int8" else s["q"].view(torch.uint8).index_select(0, source[begin:end]).view(torch.float8_e4m3fn)
            a = a.double() * s["s"].double().index_select(0, source[begin:end])[:, None]
            part = a @ (s["w"][e].double() * s["ws"][e].double()[:, None]).t()
            out[begin:end] = part if s["bias"] is None else part + s["bias"][e].double()
        begin = end
    return out
