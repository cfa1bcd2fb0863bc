"""quantize_mxfp4, dequantize_mxfp4, mxfp4_matmul, qk_norm_rope and rotary_table without a GPU: the calls their contracts
accept and refuse (on meta tensors; tests/test_gpu_four_bit_contract.py makes the same calls on the device), the wrappers' and the
module's own refusals, the scales' layout, the frequencies, and the C ABI's checks, which fail before any HIP call."""
import math

import pytest
import torch
from torch import nn

from test_experts_cpu import Make, call, none, outcome
from xgen_amd import _native as N
from xgen_amd.config import QuantLayerConfig
from xgen_amd.operator import matmul, mxfp4, runtime
from xgen_amd.operator import qk_norm_rope as qk
from xgen_amd.ops import xops

BF, HF, F32, F64, U8, I32, I64 = (torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.uint8, torch.int32, torch.int64)


def quantize(x=lambda t: t(5, 96), rounding=0):
    return lambda t: xops.quantize_mxfp4(x(t), rounding)


def dequantize(codes=lambda t: t(5, 48, dtype=U8), scales=lambda t: t(1, 6, 8, dtype=U8), out=BF):
    return lambda t: xops.dequantize_mxfp4(codes(t), scales(t), out)


def mm(a=lambda t: t(6, 48, dtype=U8), sa=lambda t: t(1, 6, 8, dtype=U8), w=lambda t: t(32, 48, dtype=U8), sw=lambda t: t(1, 32, 8, dtype=U8),
       bias=none, out=BF, act=0, res=none, gate=none, idx=none):
    return lambda t: xops.mxfp4_matmul(a(t), sa(t), w(t), sw(t), bias(t), out, act, res(t), gate(t), idx(t))


def gated(res=lambda t: t(6, 32), gate=lambda t: t(3, 32), idx=lambda t: t(2, dtype=I64), **kw):
    return mm(res=res, gate=gate, idx=idx, **kw)


def rotate(q=lambda t: t(2, 5, 4, 64), k=lambda t: t(2, 5, 2, 64), cos=lambda t: t(9, 32, dtype=F32), sin=lambda t: t(9, 32, dtype=F32),
           at=none, qw=lambda t: t(64), kw=lambda t: t(64), norm=1, eps=1e-6, inter=False):
    return lambda t: xops.qk_norm_rope(q(t), k(t), cos(t), sin(t), at(t), qw(t), kw(t), norm, eps, inter)


def table(at=lambda t: t(7, 3, dtype=I64), f=lambda t: t(20, dtype=F64), axes=lambda t: t(20, dtype=I32), factor=1.0):
    return lambda t: xops.rotary_table(at(t), f(t), axes(t), factor)


ACCEPTED = {
    "quantize": quantize(), "quantize f16": quantize(lambda t: t(5, 96, dtype=HF), 1), "quantize 1-D": quantize(lambda t: t(32)),
    "quantize 3-D": quantize(lambda t: t(2, 3, 544)), "quantize none": quantize(lambda t: t(0, 64)), "quantize transposed": quantize(lambda t: t(64, 5).t()[:, :64]),
    "quantize strided": quantize(lambda t: t(5, 200)[:, 3:99]),
    "dequantize": dequantize(), "dequantize f32": dequantize(out=F32), "dequantize f16": dequantize(out=HF),
    "dequantize 3-D": dequantize(lambda t: t(2, 3, 272, dtype=U8), lambda t: t(3, 6, 8, dtype=U8)), "dequantize none": dequantize(lambda t: t(0, 16, dtype=U8), lambda t: t(1, 0, 8, dtype=U8)),
    "mm": mm(), "mm f16": mm(out=HF, act=1, bias=lambda t: t(32, dtype=F32)), "mm bias": mm(bias=lambda t: t(32, dtype=HF)),
    "mm none": mm(a=lambda t: t(0, 48, dtype=U8), sa=lambda t: t(1, 0, 8, dtype=U8)), "mm odd": mm(a=lambda t: t(5, 48, dtype=U8)),
    "mm gated": gated(), "mm gated bias": gated(bias=lambda t: t(32)), "mm strided": mm(a=lambda t: t(6, 96, dtype=U8)[:, 16:64]),
    "rotate": rotate(), "rotate f16": rotate(q=lambda t: t(2, 5, 4, 64, dtype=HF), k=lambda t: t(2, 5, 2, 64, dtype=HF)),
    "rotate positions": rotate(at=lambda t: t(5, dtype=I64)), "rotate own positions": rotate(at=lambda t: t(2, 5, dtype=I64)),
    "rotate weights": rotate(kw=lambda t: t(64, dtype=F32)), "rotate one weight": rotate(qw=none), "rotate no norm": rotate(qw=none, kw=none, norm=-1),
    "rotate layer": rotate(norm=0, inter=True), "rotate no keys": rotate(k=lambda t: t(2, 5, 0, 64)), "rotate none": rotate(q=lambda t: t(2, 0, 4, 64), k=lambda t: t(2, 0, 2, 64)),
    "rotate views": rotate(q=lambda t: t(2, 5, 512)[..., :256].unflatten(-1, (4, 64)), k=lambda t: t(2, 5, 512)[..., 256:384].unflatten(-1, (2, 64))),
    "rotate part": rotate(cos=lambda t: t(9, 3, dtype=F32), sin=lambda t: t(9, 3, dtype=F32)), "rotate no places": rotate(cos=lambda t: t(0, 3, dtype=F32), sin=lambda t: t(0, 3, dtype=F32)),
    "table": table(), "table 1-D": table(lambda t: t(7, dtype=I64), axes=none), "table none": table(lambda t: t(0, dtype=I64), axes=none),
    "table no pairs": table(f=lambda t: t(0, dtype=F64), axes=none),
}

REFUSED = {
    "quantize f32": quantize(lambda t: t(5, 96, dtype=F32)), "quantize K": quantize(lambda t: t(5, 48)), "quantize no K": quantize(lambda t: t(5, 0)),
    "quantize rounding": quantize(rounding=2), "quantize 0-D": quantize(lambda t: t()),
    "dequantize dtype": dequantize(lambda t: t(5, 48, dtype=torch.int8)), "dequantize K": dequantize(lambda t: t(5, 24, dtype=U8)),
    "dequantize rows": dequantize(scales=lambda t: t(1, 5, 8, dtype=U8)), "dequantize blocks": dequantize(scales=lambda t: t(2, 6, 8, dtype=U8)),
    "dequantize plain scales": dequantize(scales=lambda t: t(5, 3, dtype=U8)), "dequantize out": dequantize(out=F64),
    "mm 3-D": mm(a=lambda t: t(1, 6, 48, dtype=U8)), "mm K": mm(w=lambda t: t(32, 32, dtype=U8)), "mm N": mm(w=lambda t: t(24, 48, dtype=U8), sw=lambda t: t(1, 24, 8, dtype=U8)),
    "mm no N": mm(w=lambda t: t(0, 48, dtype=U8), sw=lambda t: t(1, 0, 8, dtype=U8)), "mm a scales": mm(sa=lambda t: t(1, 4, 8, dtype=U8)),
    "mm w scales": mm(sw=lambda t: t(32, 3, dtype=U8)), "mm scale dtype": mm(sa=lambda t: t(1, 6, 8)), "mm bias size": mm(bias=lambda t: t(16)),
    "mm bias dtype": mm(bias=lambda t: t(32, dtype=F64)), "mm out": mm(out=F32), "mm activation": mm(act=2),
    "mm residual alone": mm(res=lambda t: t(6, 32)), "mm gate alone": mm(gate=lambda t: t(3, 32)), "mm no indices": gated(idx=none), "mm no gate": gated(gate=none),
    "mm gated f16": gated(out=HF), "mm gated gelu": gated(act=1), "mm residual shape": gated(res=lambda t: t(6, 16)), "mm residual f16": gated(res=lambda t: t(6, 32, dtype=HF)),
    "mm gate width": gated(gate=lambda t: t(3, 16)), "mm no table": gated(gate=lambda t: t(0, 32)), "mm seq": gated(idx=lambda t: t(4, dtype=I64)),
    "mm no seq": gated(idx=lambda t: t(0, dtype=I64)), "mm int32": gated(idx=lambda t: t(2, dtype=I32)),
    "rotate 3-D": rotate(q=lambda t: t(5, 4, 64)), "rotate f32": rotate(q=lambda t: t(2, 5, 4, 64, dtype=F32), k=lambda t: t(2, 5, 2, 64, dtype=F32)),
    "rotate mixed": rotate(k=lambda t: t(2, 5, 2, 64, dtype=HF)), "rotate seq": rotate(k=lambda t: t(2, 4, 2, 64)), "rotate width": rotate(k=lambda t: t(2, 5, 2, 32)),
    "rotate dim 60": rotate(q=lambda t: t(2, 5, 4, 60), k=lambda t: t(2, 5, 2, 60), qw=none, kw=none), "rotate dim 520": rotate(
        q=lambda t: t(2, 5, 4, 520), k=lambda t: t(2, 5, 2, 520), qw=none, kw=none), "rotate wide": rotate(cos=lambda t: t(9, 33, dtype=F32), sin=lambda t: t(9, 33, dtype=F32)),
    "rotate no pairs": rotate(cos=lambda t: t(9, 0, dtype=F32), sin=lambda t: t(9, 0, dtype=F32)), "rotate tables": rotate(sin=lambda t: t(8, 32, dtype=F32)),
    "rotate table bf16": rotate(cos=lambda t: t(9, 32), sin=lambda t: t(9, 32)), "rotate positions size": rotate(at=lambda t: t(4, dtype=I64)),
    "rotate positions int32": rotate(at=lambda t: t(5, dtype=I32)), "rotate positions shape": rotate(at=lambda t: t(1, 5, dtype=I64)), "rotate norm": rotate(norm=2),
    "rotate weight size": rotate(qw=lambda t: t(32)), "rotate weight f64": rotate(kw=lambda t: t(64, dtype=F64)), "rotate weight without norm": rotate(norm=-1),
    "rotate eps": rotate(eps=0.0), "rotate eps 1": rotate(eps=1.0),
    "table int32": table(lambda t: t(7, 3, dtype=I32)), "table 3-D": table(lambda t: t(7, 3, 1, dtype=I64)), "table no axes": table(lambda t: t(7, 0, dtype=I64)),
    "table f32": table(f=lambda t: t(20, dtype=F32)), "table f 2-D": table(f=lambda t: t(1, 20, dtype=F64)), "table axes size": table(axes=lambda t: t(19, dtype=I32)),
    "table axes int64": table(axes=lambda t: t(20, dtype=I64)), "table factor": table(factor=float("inf")),
}
NAMES = {"quantize": "quantize_mxfp4", "dequantize": "dequantize_mxfp4", "mm": "mxfp4_matmul", "rotate": "qk_norm_rope", "table": "rotary_table"}


@pytest.mark.parametrize("name", sorted(ACCEPTED))
def test_accepted(name):
    kind, got = outcome(ACCEPTED[name], "meta")
    assert kind == "accepted", got


@pytest.mark.parametrize("name", sorted(REFUSED))
def test_refused(name):
    kind, got = outcome(REFUSED[name], "meta")
    assert kind == "refused" and got.startswith(NAMES[name.split()[0]]), got


@pytest.mark.parametrize("rows,K", [(1, 32), (2, 64), (3, 256), (5, 288), (16, 544), (7, 1024)])
def test_scales_layout(rows, K):
    plain = torch.randint(0, 256, (rows, K // 32), dtype=U8, generator=torch.Generator().manual_seed(rows))
    kept = mxfp4.pack_scales(plain)
    assert kept.shape == ((K + 255) // 256, rows + rows % 2, 8)
    for r in range(rows):
        for b in range(K // 32):
            i = b % 8
            assert kept[b // 8, r, i % 2 * 4 + i // 2] == plain[r, b]
    assert int((kept != 0).sum()) == int((plain != 0).sum())  # zeros elsewhere
    assert torch.equal(mxfp4.unpack_scales(kept, rows, K), plain)
    assert torch.equal(mxfp4.pack_scales(plain.view(torch.float8_e8m0fnu)), kept)


def test_layout_refusals():
    with pytest.raises(ValueError, match="pack_scales"):
        mxfp4.pack_scales(torch.zeros(3, 4))
    with pytest.raises(ValueError, match="pack_scales"):
        mxfp4.pack_scales(torch.zeros(3, dtype=U8))
    for rows, K in ((3, 256), (4, 288), (4, 40)):
        with pytest.raises(ValueError, match="unpack_scales"):
            mxfp4.unpack_scales(torch.zeros(1, 6, 8, dtype=U8), rows, K)


def test_wrappers_refuse():
    t = Make("meta")
    grad = torch.zeros((2, 6, 64), dtype=BF, device="meta", requires_grad=True)
    with pytest.raises(ValueError, match="inference-only"):
        mxfp4.quantize_mxfp4(grad)
    with pytest.raises(ValueError, match="rounding"):
        mxfp4.quantize_mxfp4(t(2, 64), rounding="nearest")
    codes, scales = mxfp4.quantize_mxfp4(t(2, 3, 64))
    assert codes.shape == (2, 3, 32) and scales.shape == (1, 6, 8)
    w, ws = mxfp4.quantize_mxfp4(t(32, 64))
    assert mxfp4.mxfp4_matmul(codes, scales, w, ws).shape == (2, 3, 32)
    assert mxfp4.mxfp4_matmul(codes[:, :0], scales[:, :0], w, ws).shape == (2, 0, 32)
    with pytest.raises(ValueError, match="activation"):
        mxfp4.mxfp4_matmul(codes, scales, w, ws, activation="relu")
    with pytest.raises(ValueError, match="residual"):
        mxfp4.mxfp4_matmul(codes, scales, w, ws, residual=t(6, 32), gate_table=t(4, 32), indices=t(3, dtype=I64))
    with pytest.raises(ValueError, match="indices"):
        mxfp4.mxfp4_matmul(codes, scales, w, ws, residual=t(2, 3, 32), gate_table=t(4, 32), indices=t(2, dtype=I64))
    with pytest.raises(ValueError, match="inference-only"):
        mxfp4.mxfp4_matmul(codes, scales, w, ws, bias=torch.zeros(32, device="meta", requires_grad=True))
    assert mxfp4.mxfp4_matmul(codes, scales, w, ws, residual=t(2, 3, 32), gate_table=t(4, 32), indices=t(3, dtype=I64)).shape == (2, 3, 32)
    q, k, c = t(1, 5, 4, 64), t(1, 5, 2, 64), t(5, 32, dtype=F32)
    with pytest.raises(ValueError, match="norm must be"):
        qk.qk_norm_rope(q, k, c, c, norm="none")
    with pytest.raises(ValueError, match="layout"):
        qk.qk_norm_rope(q, k, c, c, layout="pairs")
    with pytest.raises(ValueError, match="inference-only"):
        qk.qk_norm_rope(q, k, c, c, q_weight=torch.ones(64, device="meta", requires_grad=True))
    assert [o.shape for o in qk.qk_norm_rope(q, k, c, c)] == [q.shape, k.shape]
    assert mxfp4.library_path().name == qk.library_path().name == "libxgen_amd.so"


def test_module_refuses():
    for shape in ((8, 64), (16, 48), (16, 64, 1)):
        with pytest.raises(ValueError, match="MXFP4Linear requires"):
            mxfp4.MXFP4Linear(torch.zeros(shape, dtype=BF))
    w, s = torch.zeros(16, 32, dtype=U8), torch.full((16, 2), 127, dtype=U8)
    linear = mxfp4.MXFP4Linear.from_packed(w, s)
    assert (linear.out_features, linear.in_features) == (16, 64) and linear.weight_scales.shape == (1, 16, 8)
    for bad in ((w.float(), s), (w[:8], s[:8]), (w, s[:, :1])):
        with pytest.raises(ValueError, match="from_packed requires"):
            mxfp4.MXFP4Linear.from_packed(*bad)
    for kw, match in ((dict(activation="relu"), "activation"), (dict(rounding="up"), "rounding"), (dict(bias=torch.zeros(15)), "bias")):
        with pytest.raises(ValueError, match=match):
            mxfp4.MXFP4Linear.from_packed(w, s, **kw)
    with pytest.raises(ValueError, match="input"):
        linear(torch.zeros(2, 32, dtype=BF))
    with pytest.raises(ValueError, match="input"):
        linear(torch.zeros(2, 64))
    x, r = torch.zeros(1, 2, 64, dtype=BF), torch.zeros(1, 2, 16, dtype=BF)
    with pytest.raises(ValueError, match="residual"):
        linear.forward_gate_residual(x, r[0], r[0], torch.zeros(2, dtype=I64))
    with pytest.raises(ValueError, match="no activation"):
        mxfp4.MXFP4Linear.from_packed(w, s, activation="gelu_tanh").forward_gate_residual(x, r, r[0], torch.zeros(2, dtype=I64))


def test_installer_names_its_formats():
    plain = nn.Sequential(nn.ReLU())
    assert matmul.enable_weight_quant_linear(plain, QuantLayerConfig(), dtype="mxfp4") is plain
    with pytest.raises(ValueError, match="w8a8.*mxfp4"):
        matmul.enable_weight_quant_linear(plain, QuantLayerConfig(), dtype="w4a16")


def test_features():
    for feature in ("mxfp4", "qk_norm_rope"):
        assert runtime.Kernels.SPECS[feature] is not None
        d = runtime.Diagnostics()
        assert runtime.Kernels(d).get(feature, torch.zeros(1)) is None and len(d.fallbacks) == 1


# --------------------------------------------------------------------------- frequencies
def test_plain_frequencies():
    f, factor = qk.rotary_frequencies(128, base=10000.0)
    assert f.dtype == F64 and factor == 1.0
    assert torch.allclose(f, torch.tensor([10000.0 ** (-i / 64) for i in range(64)], dtype=F64), rtol=1e-15, atol=0)
    linear, _ = qk.rotary_frequencies(128, scaling="linear", factor=4.0)
    assert torch.equal(linear, f / 4)
    raised, _ = qk.rotary_frequencies(128, scaling="base", factor=4.0)
    assert raised[0] == f[0] and abs(raised[-1] / (f[-1] / 4) - 1) < 1e-12  # the slowest pair as "linear"


@pytest.mark.parametrize("scaling", ["bands", "ramp"])
def test_blended_frequencies(scaling):
    f, _ = qk.rotary_frequencies(128)
    low, high, length, factor = 1.0, 32.0, 4096, 8.0
    g, scale = qk.rotary_frequencies(128, scaling=scaling, factor=factor, trained_length=length, low=low, high=high)
    turns = f * length / (2 * math.pi)
    ratio = f / g
    # (the ramp's ends are whole pairs: one further out)
    assert torch.allclose(ratio[turns >= high * 1.16], torch.ones((), dtype=F64), rtol=1e-14, atol=0)
    assert torch.allclose(ratio[turns <= low / 1.16], torch.full((), factor, dtype=F64), rtol=1e-14, atol=0)
    assert bool((ratio[1:] >= ratio[:-1] - 1e-14).all())
    assert scale == (1.0 if scaling == "bands" else 0.1 * math.log(factor) + 1)
    if scaling == "bands":
        i = int((turns > 10).sum())
        kept = (turns[i] - low) / (high - low)
        assert abs(g[i] - (f[i] * kept + f[i] / factor * (1 - kept))) < 1e-16


@pytest.mark.parametrize("kw", [dict(dim=5), dict(dim=0), dict(dim=8, base=1.0), dict(dim=8, factor=0.5), dict(dim=8, scaling="other"),
                                dict(dim=2, scaling="base"), dict(dim=8, scaling="bands"), dict(dim=8, scaling="ramp", trained_length=8, low=3.0, high=2.0)])
def test_frequency_refusals(kw):
    with pytest.raises(ValueError):
        qk.rotary_frequencies(**kw)


# --------------------------------------------------------------------------- the C ABI
QUANT = dict(dt=N.DTYPE_BF16, x=16, rows=5, K=96, ldx=96, rounding=0, codes=16, ldc=48, scales=16, block=48, s=None)
DEQUANT = dict(codes=16, ldc=48, scales=16, block=48, rows=5, K=96, dt=N.DTYPE_BF16, out=16, ldo=96, s=None)
MM = dict(a=16, lda=48, sa=16, ab=48, w=16, ldw=48, sw=16, wb=256, M=6, N=32, K=96, bias=None, bdt=N.DTYPE_NONE, act=0, res=16, ldr=32, gate=16, gs=32,
          rows=3, idx=16, seq=2, out=16, dt=N.DTYPE_BF16, ldo=32, s=None)
PLAIN = {**MM, **dict(res=None, gate=None, idx=None)}
ROT = dict(dt=N.DTYPE_BF16, q=16, qb=1280, qs=256, qh=64, nq=4, k=16, kb=640, ks=128, kh=64, nk=2, batch=2, seq=5, dim=64, norm=1, qw=16, kw=16,
           wdt=N.DTYPE_BF16, eps=1e-6, cos=16, sin=16, places=9, pairs=32, inter=0, at=None, pb=0, qo=16, ko=16, s=None)
TAB = dict(at=16, places=7, axes=3, f=16, axis=16, pairs=20, factor=1.0, cos=16, sin=16, s=None)
BAD, NO = N.ERR_INVALID_ARGUMENT, N.ERR_UNSUPPORTED


@pytest.mark.parametrize("fn,good,changes,status,needle", [
    ("xgen_mxfp4_quantize", QUANT, dict(dt=N.DTYPE_F32), BAD, b"input dtype"), ("xgen_mxfp4_quantize", QUANT, dict(rounding=2), BAD, b"rounding"),
    ("xgen_mxfp4_quantize", QUANT, dict(rows=-1), BAD, b"bad shape"), ("xgen_mxfp4_quantize", QUANT, dict(K=48, ldx=48), NO, b"multiple of 32"),
    ("xgen_mxfp4_quantize", QUANT, dict(ldx=64), BAD, b"leading"), ("xgen_mxfp4_quantize", QUANT, dict(ldc=32), BAD, b"leading"),
    ("xgen_mxfp4_quantize", QUANT, dict(block=40), BAD, b"cover"), ("xgen_mxfp4_quantize", QUANT, dict(block=56), NO, b"16-byte"),
    ("xgen_mxfp4_quantize", QUANT, dict(x=24), NO, b"aligned"), ("xgen_mxfp4_quantize", QUANT, dict(ldx=100), NO, b"aligned"),
    ("xgen_mxfp4_quantize", QUANT, dict(codes=None), BAD, b"null"), ("xgen_mxfp4_quantize", QUANT, dict(scales=20), NO, b"aligned"),
    ("xgen_mxfp4_quantize", QUANT, dict(K=1 << 30, ldx=1 << 30, ldc=1 << 29), NO, b"too many"), ("xgen_mxfp4_quantize", QUANT, dict(rows=1 << 40, block=1 << 44), NO, b"too many"),
    ("xgen_mxfp4_dequantize", DEQUANT, dict(dt=N.DTYPE_I8), BAD, b"output dtype"), ("xgen_mxfp4_dequantize", DEQUANT, dict(ldo=64), BAD, b"leading"),
    ("xgen_mxfp4_dequantize", DEQUANT, dict(ldo=100), NO, b"aligned"), ("xgen_mxfp4_dequantize", DEQUANT, dict(out=None), BAD, b"null"),
    ("xgen_mxfp4_matmul", MM, dict(M=-1), BAD, b"bad shape"), ("xgen_mxfp4_matmul", MM, dict(K=80), NO, b"multiple of 32"), ("xgen_mxfp4_matmul", MM, dict(N=24), NO, b"multiples of 16"),
    ("xgen_mxfp4_matmul", MM, dict(ab=32), BAD, b"cover"), ("xgen_mxfp4_matmul", MM, dict(wb=248), BAD, b"cover"), ("xgen_mxfp4_matmul", MM, dict(ab=56), NO, b"16-byte"),
    ("xgen_mxfp4_matmul", MM, dict(sw=24), NO, b"16-byte"), ("xgen_mxfp4_matmul", MM, dict(sa=None), BAD, b"null"), ("xgen_mxfp4_matmul", MM, dict(a=None), BAD, b"null"),
    ("xgen_mxfp4_matmul", MM, dict(lda=32), BAD, b"leading"), ("xgen_mxfp4_matmul", MM, dict(ldw=56), NO, b"aligned"), ("xgen_mxfp4_matmul", PLAIN, dict(act=2), BAD, b"activation"),
    ("xgen_mxfp4_matmul", PLAIN, dict(dt=N.DTYPE_F32), BAD, b"output dtype"), ("xgen_mxfp4_matmul", PLAIN, dict(bias=16), BAD, b"bias dtype"),
    ("xgen_mxfp4_matmul", MM, dict(act=1), BAD, b"gated residual"), ("xgen_mxfp4_matmul", MM, dict(dt=N.DTYPE_F16), BAD, b"gated residual"),
    ("xgen_mxfp4_matmul", MM, dict(gate=None), BAD, b"null"), ("xgen_mxfp4_matmul", MM, dict(seq=4), BAD, b"gated residual"), ("xgen_mxfp4_matmul", MM, dict(rows=0), BAD, b"gated residual"),
    ("xgen_mxfp4_matmul", PLAIN, dict(N=1 << 20, K=1 << 13, lda=1 << 12, ldw=1 << 12, wb=1 << 23, ldo=1 << 20), NO, b"2 GiB"),
    ("xgen_qk_norm_rope", ROT, dict(dt=N.DTYPE_F32), BAD, b"dtype"), ("xgen_qk_norm_rope", ROT, dict(pairs=33), BAD, b"bad shape"), ("xgen_qk_norm_rope", ROT, dict(pairs=0), BAD, b"bad shape"),
    ("xgen_qk_norm_rope", ROT, dict(nq=-1), BAD, b"bad shape"), ("xgen_qk_norm_rope", ROT, dict(dim=68), NO, b"multiple of 8"), ("xgen_qk_norm_rope", ROT, dict(dim=520), NO, b"multiple of 8"),
    ("xgen_qk_norm_rope", ROT, dict(norm=2), BAD, b"norm kind"), ("xgen_qk_norm_rope", ROT, dict(norm=-1), BAD, b"weights"), ("xgen_qk_norm_rope", ROT, dict(wdt=N.DTYPE_I8), BAD, b"weights"),
    ("xgen_qk_norm_rope", ROT, dict(eps=0.0), BAD, b"eps"), ("xgen_qk_norm_rope", ROT, dict(eps=float("nan")), BAD, b"eps"), ("xgen_qk_norm_rope", ROT, dict(k=None), BAD, b"null"),
    ("xgen_qk_norm_rope", ROT, dict(cos=None), BAD, b"null"), ("xgen_qk_norm_rope", ROT, dict(q=24), NO, b"aligned"), ("xgen_qk_norm_rope", ROT, dict(ko=24), NO, b"aligned"),
    ("xgen_qk_norm_rope", ROT, dict(ks=132), NO, b"multiples of 8"), ("xgen_qk_norm_rope", ROT, dict(batch=1 << 20, seq=1 << 20), NO, b"too many"),
    ("xgen_rotary_table", TAB, dict(axes=0), BAD, b"bad shape"), ("xgen_rotary_table", TAB, dict(f=None), BAD, b"null"), ("xgen_rotary_table", TAB, dict(places=1 << 30), NO, b"2^31"),
])
def test_c_entry_checks(built_library, fn, good, changes, status, needle):
    L = N.lib()
    assert call(fn, good, **changes)(L) == status, L.xgen_last_error()
    assert needle in L.xgen_last_error()


def test_c_entries_without_work(built_library):
    L = N.lib()
    assert call("xgen_mxfp4_quantize", QUANT, rows=0, x=None, codes=None, scales=None)(L) == N.OK
    assert call("xgen_mxfp4_dequantize", DEQUANT, rows=0, out=None, codes=None, scales=None)(L) == N.OK
    assert call("xgen_mxfp4_matmul", PLAIN, M=0, a=None, sa=None, w=None, sw=None, out=None)(L) == N.OK
    assert call("xgen_qk_norm_rope", ROT, seq=0, q=None, k=None, qo=None, ko=None)(L) == N.OK
    assert call("xgen_qk_norm_rope", ROT, nq=0, nk=0, q=None, k=None, qo=None, ko=None)(L) == N.OK
    assert call("xgen_rotary_table", TAB, places=0, at=None, cos=None, sin=None)(L) == N.OK
