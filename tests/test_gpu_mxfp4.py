"""MXFP4 rows and their product against plain implementations in 64 bits.

Packed rows are compared exactly: x / 2^E rounds nothing, so every byte is determined.  Tolerance of a product:
each step of 64 k adds its terms to the sum in one operation, whose error is taken as at most 2^-22 of the magnitudes it
adds (measured on random operands of any scales: 2^-23.0), so ceil(K / 64) * 2^-22 * sum |a w| in all; the bias another
2^-24, and the output half a step of its type."""
import ctypes

import pytest
import torch

import xgen_amd  # noqa: F401
from xgen_amd import _native as N
from xgen_amd.operator.mxfp4 import MXFP4Linear, dequantize_mxfp4, mxfp4_matmul, pack_scales, quantize_mxfp4, unpack_scales

pytestmark = pytest.mark.gpu
BF, HF, F32, U8 = torch.bfloat16, torch.float16, torch.float32, torch.uint8
VALUES = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)


def plain_quantize(x, rounding):
    """(codes [rows, K/2], scale bytes [rows, K/32]) on the CPU, by comparison with every code's borders."""
    v = x.double().cpu().reshape(x.shape[0], -1, 32)
    most = v.abs().amax(2)
    bad = ~torch.isfinite(most)
    most = torch.where(bad, torch.ones_like(most), most)
    mantissa, exponent = torch.frexp(most)
    e = exponent.double() - 3 + (mantissa > 0.75).double() * (rounding == "ceil")
    e = torch.where(most == 0, torch.full_like(e, -127.0), e).clamp(min=-127)
    y = torch.nan_to_num(v) * torch.exp2(-e)[..., None]
    distance = (y.abs()[..., None] - VALUES[:8]).abs()
    code = distance.argmin(-1)  # ties: the lower index, made even below
    up = (code + 1).clamp(max=7)
    tie = distance.gather(-1, up[..., None]).squeeze(-1) == distance.gather(-1, code[..., None]).squeeze(-1)
    code = torch.where(tie & (code % 2 == 1) & (code < 7), up, code)
    code = code + 8 * torch.signbit(y).long()
    code = torch.where(bad[..., None], torch.zeros_like(code), code).reshape(x.shape[0], -1)
    byte = torch.where(bad, torch.full_like(e, 255.0), e + 127)
    return (code[:, 0::2] | (code[:, 1::2] << 4)).to(U8), byte.to(U8)


def plain_values(codes, scales):
    """float64 [rows, K] of codes and scale bytes [rows, K/32]."""
    c = codes.cpu().long()
    v = VALUES[torch.stack([c & 15, c >> 4], -1).reshape(c.shape[0], -1)].reshape(c.shape[0], -1, 32)
    s = scales.cpu().double()
    return (v * torch.where(s == 255, torch.full_like(s, torch.nan), torch.exp2(s - 127))[..., None]).reshape(c.shape[0], -1)


def check_rows(cuda, x, rounding):
    codes, scales = quantize_mxfp4(x.to(cuda), rounding=rounding)
    want = plain_quantize(x.reshape(-1, x.shape[-1]), rounding)
    assert codes.dtype == scales.dtype == U8 and codes.shape == (*x.shape[:-1], x.shape[-1] // 2)
    assert torch.equal(codes.cpu().reshape(want[0].shape), want[0])
    assert torch.equal(scales.cpu(), pack_scales(want[1]))  # the padding's zeros too
    return codes, scales


def rows(g, r, k, dtype=BF, spread=6):
    """Blocks of magnitudes over 2^-spread .. 2^spread."""
    x = torch.randn((r, k // 32, 32), generator=g) * torch.exp2(torch.randint(-spread, spread + 1, (r, k // 32, 1), generator=g).float())
    return x.reshape(r, k).to(dtype)


# ----------------------------------------------------------------------------- quantize, dequantize
@pytest.mark.parametrize("rounding", ["floor", "ceil"])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("r,k", [(1, 32), (2, 64), (3, 224), (5, 256), (16, 288), (17, 512), (33, 544), (70, 5376)])
def test_rows(cuda, r, k, dtype, rounding):
    g = torch.Generator().manual_seed(r + k)
    check_rows(cuda, rows(g, r, k, dtype), rounding)


@pytest.mark.parametrize("rounding", ["floor", "ceil"])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_every_value_under_every_scale(cuda, dtype, rounding):
    """Each block: one 16-bit pattern as its largest, and 31 smaller ones around the codes' borders or at random."""
    g = torch.Generator().manual_seed(3)
    top = torch.arange(1 << 15, dtype=torch.int32).to(torch.int16).view(dtype)[:, None]
    factors = torch.cat([torch.tensor([0., -0., .25, .75, 1.25, 1.75, 2.5, 3.5, 5., 6., -.25, -.75, -2.5, -5., -6.]) / 8, torch.rand(16, generator=g) * 2 - 1])
    x = torch.cat([top, torch.nan_to_num(top.double() * factors, nan=0.0, posinf=1.0, neginf=-1.0).to(dtype)], 1)
    x[:, 1:] = torch.where(torch.isfinite(x[:, 1:]), x[:, 1:], torch.zeros((), dtype=dtype))
    sign = torch.where(torch.rand((len(x), 1), generator=g) < 0.5, -1, 1).to(dtype)
    check_rows(cuda, (x * sign).reshape(-1, 256), rounding)


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_blocks_with_inf_or_nan(cuda, bad):
    x = rows(torch.Generator().manual_seed(1), 4, 128)
    x[1, 37] = bad
    codes, scales = check_rows(cuda, x, "floor")
    back = dequantize_mxfp4(codes, scales)
    assert torch.isnan(back[1, 32:64]).all() and torch.isfinite(back).sum() == 4 * 128 - 32


def test_views(cuda):
    g = torch.Generator().manual_seed(5)
    base = rows(g, 12, 320).to(cuda)
    for x in (base[:, 32:288], base[::3, :96], base[:, 3:259], base.t()[:288 // 32 * 32, :].contiguous().t()[:, :288], base[None, :, :64],
              base.reshape(3, 4, 320)[:, 1:3, :256], base[:1].expand(5, 320)):
        codes, scales = quantize_mxfp4(x)
        want = quantize_mxfp4(x.contiguous())
        assert torch.equal(codes, want[0]) and torch.equal(scales, want[1])
    assert quantize_mxfp4(base[:0])[0].shape == (0, 160)


@pytest.mark.parametrize("dtype", [BF, HF, F32])
def test_every_code_and_scale(cuda, dtype):
    codes = torch.arange(256, dtype=torch.int32).to(U8).reshape(1, 256).repeat(16, 1).reshape(16, 256)  # 16 rows of 512 values: every byte
    scales = torch.arange(256, dtype=torch.int32).to(U8).reshape(16, 16)
    for shift in range(16):  # every block of codes with every scale
        s = scales.roll(shift, 1)
        got = dequantize_mxfp4(codes.to(cuda), pack_scales(s).to(cuda), dtype=dtype).cpu()
        want = plain_values(codes, s).float().to(dtype)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got, nan=0.0), torch.nan_to_num(want, nan=0.0)), shift


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("r,k", [(1, 32), (5, 288), (17, 544)])
def test_values(cuda, r, k, dtype):
    x = rows(torch.Generator().manual_seed(r), r, k).to(cuda)
    codes, scales = quantize_mxfp4(x)
    want = plain_values(codes, unpack_scales(scales, r, k))
    got = dequantize_mxfp4(codes.reshape(1, r, -1), scales, dtype=dtype)
    assert got.shape == (1, r, k) and torch.equal(got.cpu()[0], want.to(dtype))
    pad = torch.nn.functional.pad(codes, (0, 32))[:, :k // 2]  # rows apart
    assert torch.equal(dequantize_mxfp4(pad, scales, dtype=dtype), got[0])


def test_quantized_values_are_fixed_points(cuda):
    """A block's values quantize to themselves wherever its largest code is 4 or 6 (or 3 with the least scale)."""
    x = rows(torch.Generator().manual_seed(2), 40, 512).to(cuda)
    for rounding in ("floor", "ceil"):
        once = dequantize_mxfp4(*quantize_mxfp4(x, rounding=rounding))
        assert torch.equal(dequantize_mxfp4(*quantize_mxfp4(once, rounding=rounding)), once)


# ----------------------------------------------------------------------------- product
def packed(g, r, k, scale=1.0, rounding="ceil", spread=3):
    return quantize_mxfp4((rows(g, r, k, spread=spread) * scale).cuda(), rounding=rounding)


def values(p, r, k):
    return plain_values(p[0].reshape(r, -1), unpack_scales(p[1], r, k))


def gelu(y):
    return y / (1 + torch.exp(-2 * (2 / torch.pi) ** 0.5 * (y + 0.044715 * y ** 3)))


def check_product(a, w, m, n, k, bias=None, dtype=BF, activation=None, got=None):
    av, wv = values(a, m, k), values(w, n, k)
    y = av @ wv.t()
    error = -(-k // 64) * 2.0 ** -22 * (av.abs() @ wv.abs().t())
    if bias is not None:
        y = y + bias.double().cpu()
        error = error + 2.0 ** -24 * y.abs()
    half = torch.finfo(dtype).eps / 2
    if activation:
        # rounded before and after; |gelu'| <= 1.13, its own arithmetic 16 * 2^-24 of |y|
        error = 1.13 * (error + half * y.abs()) + 2.0 ** -20 * y.abs() + 1e-30
        y = gelu(y)
    if got is None:
        got = mxfp4_matmul(*a, *w, bias=bias, out_dtype=dtype, activation=activation)
    assert got.dtype == dtype and tuple(got.shape) == (m, n)
    error = error + half * (y.abs() + error) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (got.double().cpu() - y).abs() - error
    assert bool((off <= 0).all()), (float(off.max()), divmod(int(off.argmax()), n))
    return got


@pytest.mark.parametrize("m,n,k", [(1, 16, 32), (1, 272, 288), (2, 48, 64), (3, 2048, 96), (17, 80, 256), (31, 64, 1056), (33, 528, 512), (129, 272, 544),
                                   (257, 144, 2048), (501, 1024, 1120), (300, 2048, 5376), (1955, 528, 320)])
def test_product(cuda, m, n, k):
    g = torch.Generator().manual_seed(m + n + k)
    check_product(packed(g, m, k), packed(g, n, k, 0.02), m, n, k)


@pytest.mark.parametrize("dtype,bias,activation", [(BF, BF, None), (HF, HF, "gelu_tanh"), (BF, F32, "gelu_tanh"), (HF, None, None), (BF, HF, None)])
@pytest.mark.parametrize("m,n,k", [(5, 96, 160), (200, 400, 768), (700, 2048, 512)])
def test_epilogues(cuda, m, n, k, dtype, bias, activation):
    g = torch.Generator().manual_seed(m)
    b = None if bias is None else torch.randn(n, generator=g).to(bias).to(cuda)
    check_product(packed(g, m, k, spread=0), packed(g, n, k, 0.05, spread=0), m, n, k, b, dtype, activation)


def tile(m, n, k, gated=False):
    fn = ctypes.CDLL(str(N.library_path())).xgen_gemm_tile_choice
    fn.restype, fn.argtypes = ctypes.c_int, [ctypes.c_int] + [ctypes.c_int64] * 3 + [ctypes.c_int] * 2 + [ctypes.POINTER(ctypes.c_int)]
    cols = ctypes.c_int()
    return fn(3, m, n, k // 2, int(gated), 0, ctypes.byref(cols)), cols.value


def tile_shapes(gated=False):
    """The smallest ragged shape that runs on each tile."""
    found = {}
    for m in (1, 30, 61, 125, 251, 501, 1003, 1955, 3906, 7811):
        for n in (1040, 2064, 5392, 14352):
            for k in (96, 2080, 7136):
                t = tile(m, n, k, gated)
                if t not in found or m * n * k < found[t][0] * found[t][1] * found[t][2]:
                    found[t] = (m, n, k)
    return found


@pytest.mark.parametrize("gated", [False, True])
def test_every_tile(cuda, gated):
    """Every tile a call can run on, on a shape that is no multiple of it, against the product of a sample of its rows."""
    g = torch.Generator().manual_seed(8)
    shapes = tile_shapes(gated)
    assert (256, 256) in shapes and len(shapes) >= 4, shapes
    for t, (m, n, k) in sorted(shapes.items()):
        print("tile", t, "of", (m, n, k), flush=True)
        a, w = packed(g, m, k), packed(g, n, k, 0.02)
        at = torch.cat([torch.arange(min(m, 40)), torch.randperm(m, generator=g)[:60], torch.arange(max(0, m - 40), m)]).unique()
        part = (a[0][at.to(cuda)], pack_scales(unpack_scales(a[1], m, k)[at.to(cuda)]))
        if gated:
            res, gate, idx = gated_inputs(g, cuda, m, n, 7, m)
            got = mxfp4_matmul(*a, *w, residual=res, gate_table=gate, indices=idx)
            check_gated(part, w, len(at), n, k, None, res[at.to(cuda)], gate, idx[at.to(cuda)], got[at.to(cuda)])
        else:
            got = mxfp4_matmul(*a, *w)
            check_product(part, w, len(at), n, k, got=got[at.to(cuda)])


def test_rows_do_not_depend_on_their_company(cuda):
    """A row's result is the same bits whatever tile its call runs on."""
    g = torch.Generator().manual_seed(4)
    k, n = 1184, 2048
    a, w = packed(g, 2500, k), packed(g, n, k, 0.02)
    whole, sc = mxfp4_matmul(*a, *w), unpack_scales(a[1], 2500, k)
    for first, m in ((0, 1), (10, 16), (1000, 100), (700, 500), (1, 1300)):
        part = mxfp4_matmul(a[0][first:first + m], pack_scales(sc[first:first + m]), *w)
        assert torch.equal(part.view(torch.int16), whole[first:first + m].view(torch.int16)), (first, m)


def gated_inputs(g, cuda, m, n, t, seq):
    res = torch.randn((m, n), generator=g).to(BF).to(cuda)
    gate = torch.randn((t, n), generator=g).to(BF).to(cuda)
    return res, gate, torch.randint(0, t, (seq,), generator=g).to(cuda)


def check_gated(a, w, m, n, k, bias, res, gate, idx, got):
    """bf16(r + bf16(bf16(y) * gate)): three roundings of half a step each."""
    av, wv = values(a, m, k), values(w, n, k)
    y = av @ wv.t() + (0 if bias is None else bias.double().cpu())
    error = -(-k // 64) * 2.0 ** -22 * (av.abs() @ wv.abs().t()) + 2.0 ** -24 * y.abs()
    t = gate.double().cpu()[idx.cpu().repeat(m // len(idx))]
    half = 2.0 ** -8
    error = (error + half * (y.abs() + error)) * t.abs() * (1 + half) + half * (y * t).abs() * 1.01
    want = res.double().cpu() + y * t
    error = error + half * (want.abs() + error) + 1e-38
    off = (got.double().cpu() - want).abs() - error
    assert bool((off <= 0).all()), float(off.max())


@pytest.mark.parametrize("batch,seq,n,k,biased", [(1, 5, 96, 160, True), (3, 40, 272, 320, False), (2, 501, 1024, 1056, True)])
def test_gated_residual(cuda, batch, seq, n, k, biased):
    g = torch.Generator().manual_seed(seq)
    m = batch * seq
    a, w = packed(g, m, k), packed(g, n, k, 0.02)
    bias = torch.randn(n, generator=g).to(BF).to(cuda) if biased else None
    res, gate, idx = gated_inputs(g, cuda, m, n, 6, seq)
    got = mxfp4_matmul(a[0].reshape(batch, seq, -1), a[1], *w, bias=bias, residual=res.reshape(batch, seq, n), gate_table=gate, indices=idx)
    assert got.shape == (batch, seq, n)
    check_gated(a, w, m, n, k, bias, res, gate, idx, got.reshape(m, n))
    idx[2] = 6
    idx[3] = -1
    bad = mxfp4_matmul(*a, *w, bias=bias, residual=res, gate_table=gate, indices=idx).reshape(batch, seq, n)
    assert torch.isnan(bad[:, 2:4]).all()
    keep = [i for i in range(seq) if i not in (2, 3)]
    assert torch.equal(bad[:, keep], got[:, keep])


def test_nan_blocks_make_their_rows_nan(cuda):
    g = torch.Generator().manual_seed(6)
    for m, n, k in ((40, 64, 96), (1, 64, 96), (700, 2048, 544)):
        a, w = packed(g, m, k), packed(g, n, k, 0.02)
        good = mxfp4_matmul(*a, *w)
        sa, sw = unpack_scales(a[1], m, k), unpack_scales(w[1], n, k)
        sa[0, k // 32 - 1] = 255
        sw[5, 0] = 255
        bad = mxfp4_matmul(a[0], pack_scales(sa), w[0], pack_scales(sw))
        assert torch.isnan(bad[0]).all() and torch.isnan(bad[:, 5]).all()
        rest = [i for i in range(n) if i != 5]
        assert torch.equal(bad[1:, rest], good[1:, rest])


def test_scales_over_the_whole_range(cuda):
    """Products of scales up to 2^120 and down to 2^-120 in one row, results within fp32."""
    g = torch.Generator().manual_seed(9)
    m, n, k = 40, 48, 256
    a, w = packed(g, m, k, spread=0), packed(g, n, k, spread=0)
    shift = torch.randint(-60, 61, (k // 32,), generator=g)
    sa, sw = unpack_scales(a[1], m, k).cpu().int() + shift, unpack_scales(w[1], n, k).cpu().int() - shift
    a = (a[0], pack_scales(sa.to(U8)).to(cuda))
    w = (w[0], pack_scales(sw.to(U8)).to(cuda))
    check_product(a, w, m, n, k)


def test_operand_views(cuda):
    """Rows apart, a base off 16 bytes, scales that are a view: the same bits as contiguous operands."""
    g = torch.Generator().manual_seed(10)
    m, n, k = 37, 96, 288
    a, w = packed(g, m, k), packed(g, n, k, 0.02)
    want = mxfp4_matmul(*a, *w)
    far = torch.zeros((m, 400), dtype=U8, device=cuda)
    for at in (0, 16, 7):
        far[:, at:at + k // 2] = a[0]
        assert torch.equal(mxfp4_matmul(far[:, at:at + k // 2], a[1], *w), want)
    odd = torch.zeros(a[1].numel() + 3, dtype=U8, device=cuda)[3:].view(a[1].shape)
    odd.copy_(a[1])
    assert torch.equal(mxfp4_matmul(a[0], odd, w[0].t().contiguous().t(), w[1]), want)
    bias = torch.randn(n + 1, generator=g).to(BF).to(cuda)
    assert torch.equal(mxfp4_matmul(*a, *w, bias=bias[1:]), mxfp4_matmul(*a, *w, bias=bias[1:].clone()))
    assert mxfp4_matmul(a[0][:0], a[1][:, :0], *w).shape == (0, n)


def test_output_past_32_bit_offsets(cuda):
    """An output above 2 GiB runs in chunks of rows: rows around every border as a call of their own gives them."""
    m, n, k = 66050, 16384, 64
    g = torch.Generator(device=cuda).manual_seed(11)
    a = (torch.randint(0, 256, (m, k // 2), generator=g, device=cuda, dtype=U8), pack_scales(torch.randint(120, 130, (m, k // 32), generator=g, device=cuda, dtype=U8)))
    w = (torch.randint(0, 256, (n, k // 2), generator=g, device=cuda, dtype=U8), pack_scales(torch.randint(120, 130, (n, k // 32), generator=g, device=cuda, dtype=U8)))
    out = mxfp4_matmul(*a, *w)
    sa = unpack_scales(a[1], m, k)
    for first in (0, 32768 - 300, 65536 - 300, m - 300):
        last = min(m, first + 600)
        assert torch.equal(out[first:last], mxfp4_matmul(a[0][first:last], pack_scales(sa[first:last]), *w)), first


def test_large_rows_past_32_bit_offsets(cuda):
    """Packed rows above 2 GiB, dense rows above 4 GiB: offsets past 32 bits in both directions."""
    r, k = 300001, 14336
    x = torch.zeros((r, k), dtype=BF, device=cuda)
    g = torch.Generator().manual_seed(12)
    at = torch.tensor([0, 1, 149796, 149797, 299593, 299594, r - 2, r - 1])
    some = rows(g, len(at), k)
    x[at.to(cuda)] = some.to(cuda)
    codes, scales = quantize_mxfp4(x)
    want = plain_quantize(some, "floor")
    assert torch.equal(codes[at.to(cuda)].cpu(), want[0])
    assert torch.equal(unpack_scales(scales, r, k)[at.to(cuda)].cpu(), want[1])
    del x
    back = dequantize_mxfp4(codes, scales)
    assert torch.equal(back[at.to(cuda)].cpu(), plain_values(*want).to(BF))


# ----------------------------------------------------------------------------- module
def test_module(cuda):
    g = torch.Generator().manual_seed(13)
    weight, bias = (torch.randn((96, 160), generator=g) * 0.02).to(BF), torch.randn(96, generator=g).to(BF)
    linear = MXFP4Linear(weight, bias)
    assert linear.weight.device.type == "cpu"
    linear = linear.to(cuda)
    x = rows(g, 14, 160).reshape(2, 7, 160).to(cuda)
    out = linear(x)
    assert out.shape == (2, 7, 96) and out.dtype == BF
    a, w = quantize_mxfp4(x.reshape(14, 160), rounding="ceil"), quantize_mxfp4(weight.to(cuda), rounding="ceil")
    check_product(a, w, 14, 96, 160, bias.to(cuda), got=out.reshape(14, 96))
    assert linear(x.half()).dtype == HF and linear(x[:, :0]).shape == (2, 0, 96)
    other = MXFP4Linear.from_packed(w[0], unpack_scales(w[1], 96, 160), bias.to(cuda))
    assert torch.equal(other(x), out)
    other.load_state_dict(linear.state_dict())
    res, gate, idx = gated_inputs(g, cuda, 14, 96, 5, 7)
    got = linear.forward_gate_residual(x, res.reshape(2, 7, 96), gate, idx)
    check_gated(a, w, 14, 96, 160, bias.to(cuda), res, gate, idx, got.reshape(14, 96))


def test_installed_in_a_model(cuda):
    from xgen_amd.config import QuantLayerConfig
    from xgen_amd.operator.matmul import enable_weight_quant_linear
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(64, 96), torch.nn.GELU(), torch.nn.Linear(96, 32)).to(BF)
    x = rows(torch.Generator().manual_seed(14), 5, 64).to(cuda)
    w = quantize_mxfp4(model[0].weight.data.to(cuda), rounding="ceil")
    bias = model[0].bias.data.to(cuda)
    got = enable_weight_quant_linear(model, QuantLayerConfig(), dtype="mxfp4").to(cuda)
    assert isinstance(got[0], MXFP4Linear) and isinstance(got[2], MXFP4Linear)
    check_product(quantize_mxfp4(x, rounding="ceil"), w, 5, 96, 64, bias, got=got[0](x))
    assert got(x).shape == (5, 32)


def rounded_once(cuda, g, m, n, k, form):
    """The form's rows against 64 bits, within its sums' error and half a step."""
    a, w = packed(g, m, k, spread=0), packed(g, n, k, 0.02, spread=0)
    at = torch.cat([torch.arange(min(m, 40)), torch.randperm(m, generator=g)[:60], torch.arange(max(0, m - 40), m)]).unique()
    part = (a[0][at.to(cuda)], pack_scales(unpack_scales(a[1], m, k)[at.to(cuda)]))
    av, wv = values(part, len(at), k), values(w, n, k)
    y, error = av @ wv.t(), -(-k // 64) * 2.0 ** -22 * (av.abs() @ wv.abs().t())
    if form == "gated":
        res, gate, idx = gated_inputs(g, cuda, m, n, 7, m)
        got = mxfp4_matmul(*a, *w, residual=res, gate_table=gate, indices=idx)
        t = gate.double().cpu()[idx.cpu()[at]]
        want = res.double().cpu()[at] + y * t
        error = error * t.abs() + 2.0 ** -24 * want.abs()
    elif form == "plain":
        got, want = mxfp4_matmul(*a, *w), y
    else:
        got, want = mxfp4_matmul(*a, *w, activation="gelu_tanh", out_dtype=form), gelu(y)
        error = 1.13 * error + 2.0 ** -20 * y.abs() + 1e-30
    f = torch.finfo(got.dtype)
    error = error + f.eps / 2 * (want.abs() + error) + f.smallest_normal * f.eps
    off = (got[at.to(cuda)].double().cpu() - want).abs() - error
    assert bool((off <= 0).all()), (float(off.max()), divmod(int(off.argmax()), n))


@pytest.mark.parametrize("form", ["gated", BF, HF])
def test_one_rounding(cuda, form):
    """A gated residual and GELU are formed from the sums in 32 bits, on every tile."""
    g = torch.Generator().manual_seed(12)
    for t, (m, n, k) in sorted(tile_shapes(form == "gated").items()):
        print("tile", t, "of", (m, n, k), flush=True)
        rounded_once(cuda, g, m, n, k, form)


@pytest.mark.parametrize("form", ["gated", "plain", BF])
@pytest.mark.parametrize("k", [32, 256, 288, 544, 800, 1312])
def test_short_sums_of_many_tiles(cuda, k, form):
    """One to six pairs of K on the large tiles, three tiles a workgroup: each tile's start lies among the one before's stores."""
    m, n = 7900, 5392
    assert tile(m, n, k, form == "gated") == (256, 256)
    rounded_once(cuda, torch.Generator().manual_seed(k), m, n, k, form)


def test_gated_chunks_of_odd_rows(cuda):
    """An output above 2 GiB whose chunks are whole sequences of odd length: the second one starts at an odd row of the scales
    and ends with them."""
    seq, n, k = 33025, 16384, 64
    m = 2 * seq
    g = torch.Generator(device=cuda).manual_seed(13)
    sa = torch.randint(120, 130, (m, k // 32), generator=g, device=cuda, dtype=U8)
    a = (torch.randint(0, 256, (m, k // 2), generator=g, device=cuda, dtype=U8), pack_scales(sa))
    w = (torch.randint(0, 256, (n, k // 2), generator=g, device=cuda, dtype=U8), pack_scales(torch.randint(120, 130, (n, k // 32), generator=g, device=cuda, dtype=U8)))
    res = torch.randn((m, n), generator=g, device=cuda, dtype=BF)
    gate = torch.randn((5, n), generator=g, device=cuda, dtype=BF)
    idx = torch.randint(0, 5, (seq,), generator=g, device=cuda)
    out = mxfp4_matmul(*a, *w, residual=res, gate_table=gate, indices=idx)
    for first, last in ((0, 40), (seq - 60, seq + 61), (m - 300, m), (m - 41, m), (m - 1, m)):
        at = torch.arange(first, last, device=cuda) % seq
        part = mxfp4_matmul(a[0][first:last], pack_scales(sa[first:last]), *w, residual=res[first:last], gate_table=gate, indices=idx[at])
        assert torch.equal(out[first:last], part), first


def split(m, n, k, gated):
    fn = ctypes.CDLL(str(N.library_path())).xgen_gemm_split_choice
    fn.restype, fn.argtypes = ctypes.c_int64, [ctypes.c_int64] * 3 + [ctypes.c_int]
    return fn(m, n, k // 2, int(gated))


@pytest.mark.parametrize("form", ["gated", "plain", BF])
def test_two_launches(cuda, form):
    """Rows in two launches, an odd number of them: against 64 bits, and the bits of the last rows alone."""
    m, n, k = 3911, 5376, 7200
    first = split(m, n, k, form == "gated")
    assert 0 < first < m and first % 256 == 0
    g = torch.Generator().manual_seed(14)
    rounded_once(cuda, g, m, n, k, form)
    a, w = packed(g, m, k, spread=0), packed(g, n, k, 0.02, spread=0)
    more, part_more = {}, {}
    if form == "gated":
        res, gate, _ = gated_inputs(g, cuda, m, n, 7, 1)
        idx = torch.randint(0, 7, (m,), generator=g).to(cuda)
        more = {"residual": res, "gate_table": gate, "indices": idx}
        part_more = {"residual": res[first - 100:], "gate_table": gate, "indices": idx[first - 100:]}
    elif form is BF:
        more = part_more = {"activation": "gelu_tanh"}
    part = mxfp4_matmul(a[0][first - 100:], pack_scales(unpack_scales(a[1], m, k)[first - 100:]), *w, **part_more)
    assert torch.equal(mxfp4_matmul(*a, *w, **more)[first - 100:], part)


def test_two_launches_of_sequences(cuda):
    """Seven sequences of 559 rows: the second launch's first row is no sequence's first."""
    seq, n, k = 559, 5376, 7200
    m = 7 * seq
    first = split(m, n, k, True)
    assert first and first % seq
    g = torch.Generator().manual_seed(15)
    a, w = packed(g, m, k, spread=0), packed(g, n, k, 0.02, spread=0)
    res, gate, idx = gated_inputs(g, cuda, m, n, 7, seq)
    whole = mxfp4_matmul(*a, *w, residual=res, gate_table=gate, indices=idx)
    want = mxfp4_matmul(*a, *w, residual=res, gate_table=gate, indices=idx.repeat(7))
    assert torch.equal(whole, want)
    check_gated(a, w, m, n, k, None, res, gate, idx, whole)
