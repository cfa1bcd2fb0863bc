"""grouped_matmul: each group bit for bit the product of that group alone (scaled_mm on the same operands), and the
whole against its formula in 64 bits.

Tolerances: the output is rounded once (bf16 2^-8, f16 2^-11 relative) behind two fp32 products and a sum (3 * 2^-24 of
the magnitudes).  int8 sums are exact; exact fp8 ones sum K fp32 products (K * 2^-24 of sum |a w|); the FP8
MFMA's lose less than 2^-13 of a group of 8's largest product on each of the 8, 2^-10 of sum |a w| in all.
GELU-tanh: the slope of the function is at most 1.13, its device form is off by 2^-20 of its value and argument."""
import ctypes

import pytest
import torch

import xgen_amd  # noqa: F401
from conftest import GEMM_KINDS
from xgen_amd import _native as N
from xgen_amd.operator.experts import grouped_matmul

pytestmark = pytest.mark.gpu
xops = torch.ops.xgen_amd
FP8 = torch.float8_e4m3fn
KINDS = {"int8": (torch.int8, "exact"), "fp8": (FP8, "mfma"), "fp8_exact": (FP8, "exact")}


def quantized(g, shape, dtype, cuda):
    x = torch.randn(shape, generator=g, device=cuda)
    return (x * 32).round().clamp(-127, 127).to(torch.int8) if dtype == torch.int8 else (x * 112).clamp(-448, 448).to(FP8)


def operands(cuda, kind, counts, R, Nf, K, seed=0, bias=True):
    g = torch.Generator(device=cuda).manual_seed(seed)
    dtype, G = KINDS[kind][0], len(counts)
    return dict(q=quantized(g, (R, K), dtype, cuda), scale=torch.rand((R,), generator=g, device=cuda) * 0.02,
                weight=quantized(g, (G, Nf, K), dtype, cuda), weight_scale=torch.rand((G, Nf), generator=g, device=cuda) * 2e-4,
                ends=torch.tensor(counts, device=cuda).cumsum(0).int(),
                bias=(torch.randn((G, Nf), generator=g, device=cuda) * 0.01).bfloat16() if bias else None)


def take(t, index):
    return t.view(torch.uint8)[index].view(t.dtype)


def check(cuda, kind, ops, rows=None, activation=None, out_dtype=torch.bfloat16):
    acc = KINDS[kind][1]
    out = grouped_matmul(**ops, rows=rows, activation=activation, out_dtype=out_dtype, accumulation=acc)
    q, scale, w, ws, bias = (ops[n] for n in ("q", "scale", "weight", "weight_scale", "bias"))
    M = q.shape[0] if rows is None else rows.shape[0]
    assert out.shape == (M, w.shape[1]) and out.dtype == out_dtype
    ends, begin, half = ops["ends"].tolist(), 0, torch.finfo(out_dtype).eps / 2
    for e, end in enumerate(ends):
        if end == begin:
            continue
        r = torch.arange(begin, end, device=cuda) if rows is None else rows[begin:end].long()
        a = take(q, r)
        sa = scale if scale.numel() == 1 else scale[r]
        swe = ws[e] if ws.dim() == 2 else ws[e:e + 1]
        part = out[begin:end]
        alone, _ = xops.scaled_mm(a, w[e].contiguous(), sa.contiguous(), swe.contiguous(), None if bias is None else bias[e],
                                  out_dtype, 0 if activation is None else 1, False, kind == "fp8_exact")
        assert torch.equal(part.view(torch.int16), alone.view(torch.int16)), (e, begin, end)
        if a.shape[0] * w.shape[1] <= 1 << 22:
            s = sa.double().reshape(-1, 1) * swe.double().reshape(1, -1)
            ref = (a.double() @ w[e].double().t()) * s
            mag = (a.double().abs() @ w[e].double().abs().t()) * s
            b = 0 if bias is None else bias[e].double()
            ref, loss = ref + b, {"int8": 0.0, "fp8": 2.0 ** -10, "fp8_exact": q.shape[1] * 2.0 ** -24}[kind]
            tol = loss * mag + 3 * 2.0 ** -24 * (mag + (b.abs() if bias is not None else 0))
            if activation:
                tol = 1.13 * (tol + half * ref.abs() * (1 + half)) + 2.0 ** -20 * (1 + ref.abs())
                ref = torch.nn.functional.gelu(ref, approximate="tanh")
            assert ((part.double() - ref).abs() <= half * ref.abs() + tol * (1 + half) + 2.0 ** -25).all()
        begin = end
    assert not out[begin:].any()  # behind the last group
    return out


@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("counts,Nf,K", [
    ([1], 16, 16), ([0, 1, 0], 48, 32), ([3, 0, 0, 61, 1, 31, 33], 80, 144), ([32, 32, 64], 64, 128), ([0, 0, 5], 208, 1040),
    ([129, 0, 1, 255, 257, 64], 336, 400), ([700, 5, 300], 528, 768), ([1] * 70, 96, 272), ([0] * 40 + [9] + [0] * 60, 112, 96)])
def test_ragged_groups(cuda, kind, counts, Nf, K):
    ops = operands(cuda, kind, counts, sum(counts), Nf, K, seed=Nf + K)
    check(cuda, kind, ops)
    check(cuda, kind, {**ops, "bias": None}, activation="gelu_tanh")
    check(cuda, kind, {**ops, "bias": ops["bias"].float()}, out_dtype=torch.float16)


@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("counts,Nf,K", [
    ([2500, 1, 1600], 2064, 528), ([900] * 9, 1040, 272), ([4000, 4100], 3200, 144), ([5, 6000], 4112, 80), ([60] * 200, 528, 256),
    ([150, 90, 0, 300] * 10, 1552, 400)])
def test_many_tiles(cuda, kind, counts, Nf, K):
    """Calls of more tiles than CUs, on the larger tile sizes; gathered, too."""
    M = sum(counts)
    ops = operands(cuda, kind, counts, M, Nf, K, seed=M)
    check(cuda, kind, ops)
    g = torch.Generator(device=cuda).manual_seed(1)
    check(cuda, kind, ops, rows=torch.randint(0, M, (M,), generator=g, device=cuda, dtype=torch.int32))


@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("M,R", [(50, 7), (300, 1000), (9, 1)])
def test_gathered_rows(cuda, kind, M, R):
    """rows from an activation of another length, rows repeated."""
    counts = [M // 3, 0, M - M // 3]
    ops = operands(cuda, kind, counts, R, 176, 208, seed=M)
    g = torch.Generator(device=cuda).manual_seed(2)
    check(cuda, kind, ops, rows=torch.randint(0, R, (M,), generator=g, device=cuda, dtype=torch.int32))


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_rows_behind_the_last_group(cuda, kind):
    """Fewer pairs than rows (masked tokens, another rank's experts): zeros, whatever the row index says there."""
    ops = operands(cuda, kind, [20, 7], 100, 144, 96, seed=3)
    check(cuda, kind, ops)
    rows = torch.full((100,), -1, dtype=torch.int32, device=cuda)
    rows[:27] = torch.arange(27, 0, -1, device=cuda).int()
    check(cuda, kind, ops, rows=rows)
    none = {**ops, "ends": torch.zeros_like(ops["ends"])}
    assert not grouped_matmul(**none).any()


def test_bad_rows_make_their_output_nan(cuda):
    for kind in KINDS:
        ops = operands(cuda, kind, [30, 30], 50, 64, 64, seed=4)
        rows = torch.arange(60, device=cuda).int() % 50
        clean = grouped_matmul(**ops, rows=rows, accumulation=KINDS[kind][1])
        bad = rows.clone()
        bad[3], bad[40], bad[59] = -1, 50, 2 ** 31 - 1
        got = grouped_matmul(**ops, rows=bad, accumulation=KINDS[kind][1])
        at = torch.zeros(60, dtype=torch.bool, device=cuda)
        at[[3, 40, 59]] = True
        assert torch.isnan(got[at].float()).all() and torch.equal(got[~at], clean[~at])


def test_ends_are_taken_within_the_rows(cuda):
    ops = operands(cuda, "int8", [10, 10, 10], 30, 64, 64, seed=5)
    wide = {**ops, "ends": torch.tensor([10, 20, 1 << 30], dtype=torch.int32, device=cuda)}
    assert torch.equal(grouped_matmul(**ops), grouped_matmul(**wide))
    low = {**ops, "ends": torch.tensor([-5, 20, 30], dtype=torch.int32, device=cuda)}
    ref = {**ops, "ends": torch.tensor([0, 20, 30], dtype=torch.int32, device=cuda)}
    assert torch.equal(grouped_matmul(**ref), grouped_matmul(**low))


@pytest.mark.parametrize("G", [4, 200])
def test_an_end_below_the_one_before_is_an_empty_group(cuda, G):
    """No row has two groups, whatever the ends are: across a lane's groups and across lanes."""
    given = [700 if e % 3 == 0 else 40 + e for e in range(G - 1)] + [710]
    taken = [max(given[:e + 1]) for e in range(G)]
    ops = operands(cuda, "int8", [0] * (G - 1) + [720], 720, 64, 64, seed=6)
    got, ref = ({**ops, "ends": torch.tensor(ends, dtype=torch.int32, device=cuda)} for ends in (given, taken))
    assert torch.equal(grouped_matmul(**got), grouped_matmul(**ref))
    down = {**ops, "ends": torch.tensor([700] + [0] * (G - 1), dtype=torch.int32, device=cuda)}
    flat = {**ops, "ends": torch.tensor([700] * G, dtype=torch.int32, device=cuda)}
    assert torch.equal(grouped_matmul(**down), grouped_matmul(**flat))


def test_nan_rows_stay_theirs(cuda):
    """NaN bytes (a poisoned token) reach their own rows only, in a group's last partial tile as well."""
    ops = operands(cuda, "fp8", [33, 40], 73, 64, 80, seed=6)
    clean = grouped_matmul(**ops, accumulation="mfma")
    q = ops["q"].clone()
    q.view(torch.uint8)[32], q.view(torch.uint8)[72] = 0x7F, 0xFF
    got = grouped_matmul(**{**ops, "q": q}, accumulation="mfma")
    at = torch.zeros(73, dtype=torch.bool, device=cuda)
    at[[32, 72]] = True
    assert torch.isnan(got[at].float()).all() and torch.equal(got[~at], clean[~at])


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_scales_and_strided_operands(cuda, kind):
    counts = [40, 3, 90]
    ops = operands(cuda, kind, counts, 133, 160, 128, seed=7)
    check(cuda, kind, {**ops, "scale": ops["scale"][:1]})
    check(cuda, kind, {**ops, "weight_scale": ops["weight_scale"][:, 0].contiguous()})

    def inside(t, before, after):
        big = torch.zeros((*t.shape[:-1], t.shape[-1] + before + after), dtype=torch.uint8, device=cuda)
        big[..., before:before + t.shape[-1]] = t.view(torch.uint8)
        return big.view(t.dtype)[..., before:before + t.shape[-1]]
    ref = check(cuda, kind, ops)
    for q, w in ((inside(ops["q"], 16, 32), inside(ops["weight"], 32, 16)), (inside(ops["q"], 5, 2), inside(ops["weight"], 1, 0))):
        assert torch.equal(check(cuda, kind, {**ops, "q": q, "weight": w}), ref)
    g = torch.Generator(device=cuda).manual_seed(8)
    rows = torch.randint(0, 133, (266,), generator=g, device=cuda, dtype=torch.int32)
    assert torch.equal(check(cuda, kind, {**ops, "q": inside(ops["q"], 16, 32)}, rows=rows[::2]), check(cuda, kind, ops, rows=rows[::2].contiguous()))
    one = ops["weight"][:1].view(torch.uint8).expand(3, 160, 128).view(ops["weight"].dtype)  # one weight for every group
    check(cuda, kind, {**ops, "weight": one})


def test_most_groups(cuda):
    counts = [(i * 7) % 5 for i in range(512)]
    check(cuda, "int8", operands(cuda, "int8", counts, sum(counts), 32, 64, seed=9))
    counts = [0] * 511 + [700]
    check(cuda, "fp8", operands(cuda, "fp8", counts, 700, 32, 64, seed=10))


def test_no_rows(cuda):
    ops = operands(cuda, "fp8", [0, 0], 0, 32, 64, seed=11)
    assert grouped_matmul(**ops).shape == (0, 32)
    ops = operands(cuda, "fp8", [0, 0], 4, 32, 64, seed=11)
    assert grouped_matmul(**ops, rows=torch.empty(0, dtype=torch.int32, device=cuda)).shape == (0, 32)


def test_weights_past_32_bit_offsets(cuda):
    """Six groups' weights of 768 MB: the last one's start past 2^32 bytes."""
    G, Nf, K = 6, 49152, 16384
    w = torch.zeros((G, Nf, K), dtype=torch.int8, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(12)
    w[5, -64:] = quantized(g, (64, K), torch.int8, cuda)
    q = quantized(g, (40, K), torch.int8, cuda)
    s, ws = torch.rand((40,), generator=g, device=cuda), torch.rand((G, Nf), generator=g, device=cuda) * 1e-4
    ends = torch.tensor([0, 0, 3, 3, 3, 40], dtype=torch.int32, device=cuda)
    out = grouped_matmul(q, s, w, ws, ends)
    ref, _ = xops.scaled_mm(q[3:], w[5, -64:], s[3:].clone(), ws[5, -64:].clone(), None, torch.bfloat16, 0, False)
    assert torch.equal(out[3:, -64:], ref) and not out[:3].any() and not out[:, :-64].any()


def test_outputs_past_32_bit_offsets(cuda):
    """An output of 4.9 GB and an activation of 2.4 GB (not gathered)."""
    M, Nf, K = 150000, 16384, 16384 - 16
    q = torch.zeros((M, K), dtype=torch.int8, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(13)
    q[-100:] = quantized(g, (100, K), torch.int8, cuda)
    w = quantized(g, (2, Nf, K), torch.int8, cuda)
    s, ws = torch.rand((M,), generator=g, device=cuda), torch.rand((2, Nf), generator=g, device=cuda) * 1e-4
    ends = torch.tensor([M - 50, M], dtype=torch.int32, device=cuda)
    out = grouped_matmul(q, s, w, ws, ends)
    for e, part in ((0, slice(M - 100, M - 50)), (1, slice(M - 50, M))):
        ref, _ = xops.scaled_mm(q[part], w[e], s[part].clone(), ws[e], None, torch.bfloat16, 0, False)
        assert torch.equal(out[part], ref)
    assert not out[:M - 100:997].any()
    with pytest.raises(RuntimeError, match="indexed"):
        grouped_matmul(q, s, w, ws, ends, rows=torch.zeros(4, dtype=torch.int32, device=cuda))
    assert N.lib().xgen_last_error()


def tile_of(kind, M, Nf, K, groups):
    fn = ctypes.CDLL(str(N.library_path())).xgen_grouped_tile_choice
    fn.argtypes = [ctypes.c_int] + [ctypes.c_int64] * 4 + [ctypes.POINTER(ctypes.c_int)]
    n = ctypes.c_int()
    m = fn(GEMM_KINDS[kind], M, Nf, K, groups, ctypes.byref(n))
    return m, n.value


# (groups, fewest and most rows of one, N, K): several tiles per workgroup on each tile
MANY = [(24, 10, 90, 2064, 1552), (40, 20, 300, 1552, 1040), (64, 40, 330, 2064, 656), (12, 300, 900, 2576, 1168),
        (8, 1000, 2500, 3600, 1296), (128, 5, 120, 1040, 784), (4, 1, 9, 2064, 1040), (20, 1, 70, 912, 400), (19, 300, 1200, 2320, 880), (9, 118, 354, 2912, 2048)]
TILES = {(32, 128), (64, 128), (64, 192), (128, 128), (128, 192), (256, 192), (256, 256)}


def many_counts(case):
    g = torch.Generator().manual_seed(case[3])
    counts = torch.randint(case[1], case[2] + 1, (case[0],), generator=g).tolist()
    counts[1] = 0
    return counts


@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("case", MANY)
def test_every_tile(cuda, kind, case):
    counts = many_counts(case)
    M = sum(counts)
    ops = operands(cuda, kind, counts, M, case[3], case[4], seed=M)
    check(cuda, kind, ops)
    g = torch.Generator(device=cuda).manual_seed(3)
    rows = torch.randint(0, M, (M + 40,), generator=g, device=cuda, dtype=torch.int32)
    check(cuda, kind, {**ops, "bias": None}, rows=rows, activation="gelu_tanh", out_dtype=torch.float16)


@pytest.mark.parametrize("kind", sorted(KINDS))
@pytest.mark.parametrize("most", [4, 24, 60, 110, 190])
def test_weights_past_the_last_level_cache(cuda, kind, most):
    """316 MB of weights, each read by about one tile row or by two: past the caches and through them."""
    g = torch.Generator().manual_seed(most)
    counts = torch.randint(1, most + 1, (96,), generator=g).tolist()
    counts[5] = 0
    M = sum(counts)
    ops = operands(cuda, kind, counts, M, 2064, 1600, seed=most)
    check(cuda, kind, ops)
    rows = torch.randperm(M, generator=g).to(cuda, torch.int32)
    check(cuda, kind, {**ops, "bias": None}, rows=rows, activation="gelu_tanh", out_dtype=torch.float16)


@pytest.mark.parametrize("kind", sorted(KINDS))
def test_the_cases_above_take_every_tile(cuda, kind):
    taken = {tile_of(kind, sum(many_counts(c)), c[3], c[4], c[0]) for c in MANY}
    taken |= {tile_of(kind, c["M"], c["N"], c["K"], c["G"]) for c in (dict(M=9, N=2064, K=1040, G=3), dict(M=706, N=336, K=400, G=6))}
    check(cuda, kind, operands(cuda, kind, [3, 0, 6], 9, 2064, 1040, seed=20))
    check(cuda, kind, operands(cuda, kind, [129, 0, 1, 255, 257, 64], 706, 336, 400, seed=21))
    assert taken == (TILES - {(256, 256)} if kind == "fp8_exact" else TILES), taken


def test_more_tiles_than_a_workgroup_lists_at_once(cuda):
    """70 tiles a workgroup: the list of tiles is filled again twice."""
    counts = [30000, 1, 25000, 14999]
    ops = operands(cuda, "int8", counts, 70000, 16400, 32, seed=22)
    assert tile_of("int8", 70000, 16400, 32, 4) == (256, 256)
    check(cuda, "int8", ops)
