"""The 4-bit linear path and the rotation of queries and keys: the calls that are timed and what their outputs are compared with.

Operators: MXFP4 rows (`quantize_mxfp4`, `dequantize_mxfp4`), their product (`mxfp4_matmul`), the norms of queries and keys per
head with the position rotation in one pass (`qk_norm_rope`), and the table of angles it reads (`rotary_table`).  Widths are
d = 5,376 with its 14,336-wide feed-forward and 56 heads of 128, tokens 15,624, 3,906, 1,955 and 501, as elsewhere in this package,
and generic ones.

Formulas, all in real numbers (outputs are rounded once, to their type):

  quantize    each 32 consecutive values of a row: E = floor(log2 max|x|) - 2 ("floor") or the least E with max|x| <= 6 * 2^E
              ("ceil"), -127 at least; code = the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 to |x| / 2^E (ties to the even code), signed
  dequantize  code * 2^E
  matmul      y[m, n] = sum_k a[m, k] w[n, k] + bias[n];  gelu_tanh(y), or residual + gate[i] * y with i = indices[m mod seq]
  rotate      v = norm(x) * w over each head; pairs (a, b) of its first R values, (i, i + R/2) or (2 i, 2 i + 1), become
              (a cos - b sin, b cos + a sin) with the angles of the token's position
  table       cos and sin of positions[p, axis[i]] * f[i], times a factor

Packed codes: two per byte, the even k in the low four bits.  Scales: the bytes E + 127 as [ceil(K / 256), rows rounded up to even, 8],
block i of a row's 256 values at byte (i mod 2) * 4 + i div 2.
"""
from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
TABLE_ROWS = 20
EPS = 1e-6
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MOST_FLOPS = 2 * 15624 * 14336 * 5376
MOST_VALUES = 15624 * 5376
MOST_HEADS = 15624 * 2 * 56 * 128
MOST_ANGLES = 15624 * 64


def listed():
    return [
        # a projection of two requests' new tokens, quantized on the way in
        dict(name="linear_2", op="linear", tokens=2, k=2048, n=2048, rounding="floor", bias=False, activation="none", gated=False, dtype="bf16"),
        # a small image request's square projection
        dict(name="linear_501", op="linear", tokens=501, k=5376, n=5376, rounding="ceil", bias=True, activation="none", gated=False, dtype="bf16"),
        # up-projection of eight new tokens: the weights are what is read
        dict(name="matmul_8", op="matmul", tokens=8, k=5376, n=14336, rounding="ceil", bias=False, activation="none", gated=False, dtype="f16"),
        # down-projection of a clip's token share with the gated residual behind it
        dict(name="matmul_3906", op="matmul", tokens=3906, k=14336, n=5376, rounding="ceil", bias=True, activation="none", gated=True, dtype="bf16"),
        # the largest: a 5 s clip's up-projection with its activation
        dict(name="matmul_15624", op="matmul", tokens=15624, k=5376, n=14336, rounding="floor", bias=True, activation="gelu_tanh", gated=False, dtype="bf16"),
        # rows sent in 4 bits and taken back: a small request in half precision
        dict(name="pack_501", op="pack", tokens=501, k=1024, rounding="ceil", dtype="f16"),
        # the same for a clip's activations
        dict(name="pack_15624", op="pack", tokens=15624, k=5376, rounding="floor", dtype="bf16"),
        # four requests' new tokens at far positions of their own, shared keys
        dict(name="rotate_4", op="rotate", batch=4, seq=1, heads=32, kv=8, dim=128, rotary=128, layout="half", norm="rms", weights=True, places=131072,
             own_places=True, dtype="bf16"),
        # part of each head rotated, pairs side by side, another norm, odd token count
        dict(name="rotate_1955", op="rotate", batch=2, seq=1955, heads=20, kv=20, dim=64, rotary=48, layout="interleaved", norm="layer", weights=True,
             places=4096, own_places=False, dtype="f16"),
        # a clip's queries and keys, all heads, out of the fused projection's rows
        dict(name="rotate_15624", op="rotate", batch=1, seq=15624, heads=56, kv=56, dim=128, rotary=128, layout="half", norm="rms", weights=True,
             places=15624, own_places=False, dtype="bf16"),
        # the angles of a decoding step at far positions, frequencies as scaled for a long context
        dict(name="table_4", op="table", places=4, axes=1, pairs=64, far=1000000, factor=1.1386),
        # a clip's angles, three axes
        dict(name="table_15624", op="table", places=15624, axes=3, pairs=64, far=128, factor=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "matmul", "matmul", "matmul", "pack", "pack", "rotate", "rotate", "table"])
    tokens = _log_int(rng, 1, 15624)
    dtype = rng.choice(["bf16", "bf16", "f16"])
    rounding = rng.choice(["floor", "ceil"])
    if op == "table":
        axes, pairs = rng.choice([1, 1, 2, 3]), rng.randint(4, 128)
        return dict(op=op, places=min(tokens, MOST_ANGLES // pairs), axes=axes, pairs=pairs, far=_log_int(rng, 64, 1000000),
                    factor=rng.choice([1.0, 1.1386]))
    if op == "rotate":
        dim = rng.choice([64, 128, 128, 256, 8 * rng.randint(4, 32)])
        rotary = dim if rng.random() < 0.5 else 2 * rng.randint(2, dim // 2)
        kv = rng.choice([1, 2, 4, 8, 20])
        heads = kv * rng.randint(1, max(1, 56 // kv))
        batch = rng.choice([1, 1, 2, 5])
        seq = max(1, min(tokens, MOST_HEADS // ((heads + kv) * dim)) // batch)
        return dict(op=op, batch=batch, seq=seq, heads=heads, kv=kv, dim=dim, rotary=rotary, layout=rng.choice(["half", "interleaved"]),
                    norm=rng.choice(["rms", "rms", "layer", "none"]), weights=rng.random() < 0.8, places=max(seq, rng.choice([256, 4096, 131072])),
                    own_places=rng.random() < 0.5, dtype=dtype)
    k = 32 * rng.randint(16, 448)
    if op == "pack":
        return dict(op=op, tokens=min(tokens, MOST_VALUES // k), k=k, rounding=rounding, dtype=dtype)
    n = 16 * rng.randint(32, 896)
    tokens = max(1, min(tokens, MOST_FLOPS // (2 * n * k)))
    gated = rng.random() < 0.3
    return dict(op=op, tokens=tokens, k=k, n=n, rounding=rounding, bias=rng.random() < 0.6,
                activation="none" if gated else rng.choice(["none", "gelu_tanh"]), gated=gated, dtype="bf16" if gated else dtype)


# ----------------------------------------------------------------------------- inputs
def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float16


def _randn(g, *shape, scale=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _rows(g, tokens, k, dtype):
    """Activations with a few channels far above the others, as a block's are."""
    x = _randn(g, tokens, k, dtype=dtype)
    x[:, torch.randperm(k, generator=g, device=DEV)[:max(1, k // 1000)]] *= 50
    return x


def _layout(scales):
    """Scale bytes [rows, K / 32] as the packed rows' operators keep them."""
    rows, blocks = scales.shape
    out = scales.new_zeros((rows + rows % 2, (blocks + 7) // 8 * 8))
    out[:rows, :blocks] = scales
    return out.reshape(out.shape[0], -1, 4, 2).permute(1, 0, 3, 2).reshape(-1, out.shape[0], 8).contiguous()


def _plain_quantize(x, rounding):
    """codes uint8 [rows, K / 2] and scale bytes uint8 [rows, K / 32] of finite rows."""
    v = x.float().reshape(x.shape[0], -1, 32)
    mantissa, exponent = torch.frexp(v.abs().amax(dim=2))  # in [0.5, 1) times 2^exponent
    e = exponent - 3
    if rounding == "ceil":
        e = e + (mantissa > 0.75).int()
    e = torch.where(mantissa > 0, e, -127).clamp(min=-127)
    v = torch.ldexp(v, -e[:, :, None])
    a = v.abs()
    code = torch.zeros_like(a, dtype=torch.uint8)
    for i, border in enumerate((0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)):  # between code i and i + 1; a tie goes to the even one
        code += ((a > border) if i % 2 == 0 else (a >= border)).to(torch.uint8)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).reshape(x.shape[0], -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), (e + 127).to(torch.uint8)


def _plain_values(codes, scales):
    """float32 [rows, K] of codes and scale bytes [rows, K / 32]."""
    table = torch.tensor(VALUES + tuple(-v for v in VALUES), device=codes.device)
    v = table[torch.stack([codes & 15, codes >> 4], dim=-1).reshape(codes.shape[0], -1).int()]
    return torch.ldexp(v.reshape(codes.shape[0], -1, 32), (scales.int() - 127)[:, :, None]).reshape(v.shape)


def _row_scales(scales, rows, blocks):
    """Scale bytes [rows, K / 32] out of the kept layout."""
    return scales.reshape(scales.shape[0], -1, 2, 4).permute(1, 0, 3, 2).reshape(scales.shape[1], -1)[:rows, :blocks]


def _linear_inputs(case, g):
    tokens, k, n, dtype = case["tokens"], case["k"], case["n"], _type(case)
    x = _rows(g, tokens, k, dtype)
    w = torch.randn((n, k), generator=g, device=DEV).mul_(0.02).to(torch.bfloat16)
    given = dict(x=x, w=w, bias=_randn(g, n, scale=0.01) if case["bias"] else None, residual=None, gate=None, indices=None)
    if case["gated"]:
        given.update(residual=_randn(g, tokens, n), gate=_randn(g, TABLE_ROWS, n, scale=0.5),
                     indices=torch.randint(0, TABLE_ROWS, (tokens,), generator=g, device=DEV))
    return given


def _rotate_inputs(case, g):
    batch, seq, heads, kv, dim, pairs = (case[c] for c in ("batch", "seq", "heads", "kv", "dim", "rotary"))
    pairs //= 2
    fused = _randn(g, batch, seq, (heads + 2 * kv) * dim, dtype=_type(case))  # a fused projection's rows: queries, keys, values
    q, k, _ = fused.split([heads * dim, kv * dim, kv * dim], dim=-1)
    angle = torch.arange(case["places"], dtype=torch.float64, device=DEV)[:, None] * _frequencies(pairs)
    weights = [1 + _randn(g, dim, scale=0.1, dtype=_type(case)) if case["weights"] else None for _ in range(2)]
    positions = torch.randint(0, case["places"], (batch, seq), generator=g, device=DEV) if case["own_places"] else None
    return dict(q=q.unflatten(-1, (heads, dim)), k=k.unflatten(-1, (kv, dim)), cos=angle.cos().float(), sin=angle.sin().float(),
                positions=positions, qw=weights[0], kw=weights[1])


def _frequencies(pairs):
    return 10000.0 ** (-torch.arange(pairs, dtype=torch.float64, device=DEV) / pairs)


def _inputs(case, seed):
    g, op = torch.Generator(device=DEV).manual_seed(seed), case["op"]
    if op == "rotate":
        return _rotate_inputs(case, g)
    if op == "table":
        axes, pairs = case["axes"], case["pairs"]
        return dict(positions=torch.randint(0, case["far"], (case["places"], axes), generator=g, device=DEV), f=_frequencies(pairs),
                    axis=(torch.arange(pairs, device=DEV) * axes // pairs).int())
    if op == "pack":
        return dict(x=_rows(g, case["tokens"], case["k"], _type(case)))
    return _linear_inputs(case, g)


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if case["op"] in ("linear", "matmul"):
        codes, scales = _plain_quantize(state.pop("w"), "ceil")
        state.update(wq=codes, ws=_layout(scales))
    if case["op"] == "matmul":
        codes, scales = _plain_quantize(state.pop("x"), case["rounding"])
        state.update(aq=codes, s=_layout(scales))
    return state


# ----------------------------------------------------------------------------- plain forms
def _gelu(y):
    return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))


def _plain_matmul(s):
    case = s["case"]
    blocks = case["k"] // 32
    if case["op"] == "linear":
        a = _plain_values(*_plain_quantize(s["x"], case["rounding"]))
    else:
        a = _plain_values(s["aq"], _row_scales(s["s"], case["tokens"], blocks))
    y = a @ _plain_values(s["wq"], _row_scales(s["ws"], case["n"], blocks)).t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    if case["activation"] == "gelu_tanh":
        y = _gelu(y)
    if s["residual"] is not None:
        y = s["residual"].float() + s["gate"].float()[s["indices"]] * y
    return y.to(_type(case))


def _normed(v, kind):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(dim=-1, keepdim=True)
    return v * torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + EPS)


def _plain_rotate(s):
    case, half = s["case"], s["case"]["rotary"] // 2
    places = torch.arange(case["seq"], device=s["q"].device) if s["positions"] is None else s["positions"]
    cos, sin = s["cos"][places].unsqueeze(-2), s["sin"][places].unsqueeze(-2)
    out = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        v = _normed(x.float(), case["norm"])
        if w is not None and case["norm"] != "none":
            v = v * w.float()
        turned, rest = v[..., :2 * half], v[..., 2 * half:]
        if case["layout"] == "half":
            a, b = turned[..., :half], turned[..., half:]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        else:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
        out.append(torch.cat([turned, rest], dim=-1).to(_type(case)))
    return tuple(out)


def _plain_table(s):
    angle = s["positions"].double()[:, s["axis"].long()] * s["f"]
    return (angle.cos() * s["case"]["factor"]).float(), (angle.sin() * s["case"]["factor"]).float()


# ----------------------------------------------------------------------------- the framework's operators
_API = []


def _api():
    if not _API:
        from xgen_amd.operator.mxfp4 import dequantize_mxfp4, mxfp4_matmul, quantize_mxfp4
        from xgen_amd.operator.qk_norm_rope import qk_norm_rope, rotary_table
        _API.append((quantize_mxfp4, dequantize_mxfp4, mxfp4_matmul, qk_norm_rope, rotary_table))
    return _API[0]


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        quantize, dequantize, matmul, rotate, table = _api()
        if op == "pack":
            return dequantize(*quantize(state["x"], rounding=case["rounding"]), dtype=_type(case))
        if op == "rotate":
            plain = case["norm"] == "none"
            return rotate(state["q"], state["k"], state["cos"], state["sin"], positions=state["positions"],
                          q_weight=None if plain else state["qw"], k_weight=None if plain else state["kw"],
                          norm=None if plain else case["norm"], eps=EPS, layout=case["layout"])
        if op == "table":
            return table(state["positions"], state["f"], axes=state["axis"], factor=case["factor"])
        codes, scales = quantize(state["x"], rounding=case["rounding"]) if op == "linear" else (state["aq"], state["s"])
        return matmul(codes, scales, state["wq"], state["ws"], bias=state["bias"], out_dtype=_type(case),
                      activation=None if case["activation"] == "none" else case["activation"],
                      residual=state["residual"], gate_table=state["gate"], indices=state["indices"])
    if op == "pack":
        return _plain_values(*_plain_quantize(state["x"], case["rounding"])).to(_type(case))
    if op == "rotate":
        return _plain_rotate(state)
    if op == "table":
        return _plain_table(state)
    return _plain_matmul(state)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    op = case["op"]
    packed = 17 / 32  # bytes of a value: half a byte of code, a 32nd of a scale
    if op == "table":
        size = case["places"] * case["pairs"]
        return {"bytes": 8 * case["places"] * case["axes"] + 8 * size + 12 * case["pairs"], "flops": 40 * size}
    if op == "rotate":
        tokens, heads = case["batch"] * case["seq"], case["heads"] + case["kv"]
        rows = min(tokens, case["places"]) if case["own_places"] else case["seq"]
        return {"bytes": tokens * heads * case["dim"] * 4 + rows * case["rotary"] * 4, "flops": 8 * tokens * heads * case["dim"]}
    m, k = case["tokens"], case["k"]
    if op == "pack":  # packed rows are written and read back, as what is sent is
        return {"bytes": m * k * (4 + 2 * packed), "flops": 4 * m * k}
    n = case["n"]
    given = m * k * (2 if op == "linear" else packed)
    gated = 2 * m * n + 2 * n * min(m, TABLE_ROWS) if case["gated"] else 0
    return {"bytes": given + n * k * packed + 2 * m * n + gated + (2 * n if case["bias"] else 0), "flops": 2 * m * n * k}


# ----------------------------------------------------------------------------- the definitions in 64 bits
def _exact_values(x, rounding):
    """The values that finite rows keep in 4 bits."""
    v = x.double().unflatten(1, (-1, 32))
    most = v.abs().max(dim=2, keepdim=True).values
    if rounding == "floor":
        e = torch.floor(torch.log2(most)) - 2
    else:
        e = torch.ceil(torch.log2(most / 6))
    unit = torch.exp2(e.clamp(min=-127))  # (log2(0) is -inf: a block of zeros takes the least)
    y = v / unit
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=1.0))) - 1)
    return ((torch.round(y / step) * step).clamp(-6, 6) * unit).flatten(1)


def exact(case, seed):
    s, op = _inputs(case, seed), case["op"]
    if op == "pack":
        return _exact_values(s["x"], case["rounding"])
    if op == "table":
        columns = [s["positions"][:, a].double() for a in s["axis"].tolist()]
        angle = torch.stack([c * f for c, f in zip(columns, s["f"])], dim=1)
        return case["factor"] * torch.cos(angle), case["factor"] * torch.sin(angle)
    if op == "rotate":
        r, out = case["rotary"], []
        at = torch.arange(case["seq"], device=DEV).expand(case["batch"], -1) if s["positions"] is None else s["positions"]
        c, d = (t.double().index_select(0, at.flatten()).reshape(*at.shape, 1, r // 2) for t in (s["cos"], s["sin"]))
        for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
            v = x.double()
            if case["norm"] != "none":
                if case["norm"] == "layer":
                    v = v - v.sum(-1, keepdim=True) / case["dim"]
                v = v / ((v ** 2).sum(-1, keepdim=True) / case["dim"] + EPS).sqrt()
                v = v if w is None else v * w.double()
            else:
                v = v.clone()
            first, second = (slice(0, r // 2), slice(r // 2, r)) if case["layout"] == "half" else (slice(0, r, 2), slice(1, r, 2))
            a, b = v[..., first].clone(), v[..., second].clone()
            v[..., first], v[..., second] = a * c - b * d, b * c + a * d
            out.append(v)
        return tuple(out)
    a, w = _exact_values(s["x"], case["rounding"]), _exact_values(s["w"], "ceil")
    y = torch.mm(a, w.t().contiguous())
    if s["bias"] is not None:
        y += s["bias"].double()
    if case["activation"] == "gelu_tanh":
        y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    if s["residual"] is not None:
        y = y * s["gate"].double().index_select(0, s["indices"]) + s["residual"].double()
    return y
