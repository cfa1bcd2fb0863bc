"""residual_norm, route, grouped_matmul and combine without a GPU: the calls their contracts accept and
refuse (on meta tensors; tests/test_gpu_experts_contract.py makes the same calls on the device), the wrappers' and the module's own
refusals, and the C ABI's checks, which fail before any HIP call."""
import pytest
import torch

from xgen_amd import _native as N
from xgen_amd.operator import experts as ex
from xgen_amd.operator.residual_norm import residual_norm
from xgen_amd.operator import runtime
from xgen_amd.ops import xops

BF, HF, F32, F8, I8, I32, I64 = (torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn, torch.int8, torch.int32,
                                 torch.int64)


class Make:
    def __init__(self, device):
        self.device = device

    def __call__(self, *shape, dtype=BF):
        t = torch.zeros(shape, dtype=torch.uint8 if dtype == F8 else dtype, device=self.device)
        return t.view(F8) if dtype == F8 else t


def none(t):
    return None


def norm(x=lambda t: t(2, 6, 64), y=lambda t: t(2, 6, 64), wb=lambda t: t(64), w=lambda t: t(64), gate=lambda t: t(3, 64),
         scale=lambda t: t(3, 64), shift=lambda t: t(3, 64), idx=lambda t: t(6, dtype=I64), bn=1, kind=1, a=1.0, eps=1e-5, out=BF):
    return lambda t: xops.residual_norm(x(t), y(t), wb(t), w(t), gate(t), scale(t), shift(t), idx(t), bn, kind, a, eps, out)


def route(x=lambda t: t(70, 16, dtype=F32), k=2, bias=none, scoring=0, renormalize=True, first=0, local=16):
    return lambda t: xops.route(x(t), k, bias(t), scoring, renormalize, first, local)


def grouped(a=lambda t: t(5, 32, dtype=F8), sa=lambda t: t(5, dtype=F32), w=lambda t: t(3, 48, 32, dtype=F8),
            sw=lambda t: t(3, 48, dtype=F32), ends=lambda t: t(3, dtype=I32), rows=none, bias=none, out=BF, act=0, exact=False):
    return lambda t: xops.grouped_matmul(a(t), sa(t), w(t), sw(t), ends(t), rows(t), bias(t), out, act, exact)


def combine(y=lambda t: t(12, 64), w=lambda t: t(6, 2, dtype=F32), s=lambda t: t(6, 2, dtype=I32), res=none, gate=none, idx=none):
    return lambda t: xops.expert_combine(y(t), w(t), s(t), res(t), gate(t), idx(t))


ACCEPTED = {
    "norm": norm(), "norm fp8": norm(out=F8), "norm int8": norm(out=I8), "norm layer": norm(kind=0, bn=0),
    "norm no branch norm": norm(bn=-1, wb=none), "norm bare": norm(wb=none, w=none, gate=none, scale=none, shift=none, idx=none),
    "norm f32 weights": norm(w=lambda t: t(64, dtype=F32)), "norm no gate": norm(gate=none), "norm gate only": norm(scale=none, shift=none),
    "norm empty": norm(x=lambda t: t(0, 6, 64), y=lambda t: t(0, 6, 64)), "norm widest": norm(
        x=lambda t: t(1, 2, 8192), y=lambda t: t(1, 2, 8192), wb=none, w=none, gate=none, scale=none, shift=none, idx=none),
    "norm strided indices": norm(idx=lambda t: t(12, dtype=I64)[::2]), "norm transposed": norm(x=lambda t: t(6, 2, 64).transpose(0, 1)),
    "route": route(), "route bf16": route(x=lambda t: t(70, 16)), "route f16": route(x=lambda t: t(7, 16, dtype=HF)),
    "route bias": route(bias=lambda t: t(16, dtype=F32)), "route sigmoid": route(scoring=1, renormalize=False),
    "route part": route(first=4, local=3), "route none": route(x=lambda t: t(0, 16, dtype=F32)), "route all": route(k=16),
    "route strided": route(x=lambda t: t(16, 70, dtype=F32).t()), "route most": route(x=lambda t: t(3, 512, dtype=F32), k=32, local=512),
    "grouped": grouped(), "grouped exact": grouped(exact=True), "grouped int8": grouped(a=lambda t: t(5, 32, dtype=I8), w=lambda t: t(3, 48, 32, dtype=I8)),
    "grouped rows": grouped(rows=lambda t: t(9, dtype=I32)), "grouped bias": grouped(bias=lambda t: t(3, 48, dtype=HF), out=HF, act=1),
    "grouped one scale": grouped(sa=lambda t: t(1, dtype=F32), sw=lambda t: t(3, dtype=F32)), "grouped none": grouped(a=lambda t: t(0, 32, dtype=F8), sa=lambda t: t(0, dtype=F32)),
    "grouped no rows": grouped(rows=lambda t: t(0, dtype=I32)),
    "combine": combine(), "combine f16": combine(y=lambda t: t(12, 64, dtype=HF)), "combine residual": combine(res=lambda t: t(6, 64)),
    "combine gate": combine(res=lambda t: t(6, 64), gate=lambda t: t(4, 64), idx=lambda t: t(3, dtype=I64)),
    "combine no rows": combine(y=lambda t: t(1, 64)), "combine none": combine(w=lambda t: t(0, 2, dtype=F32), s=lambda t: t(0, 2, dtype=I32)),
}

REFUSED = {
    "norm 2-D": norm(x=lambda t: t(12, 64), y=lambda t: t(12, 64)), "norm shapes": norm(y=lambda t: t(2, 6, 32)), "norm f16": norm(x=lambda t: t(2, 6, 64, dtype=HF)),
    "norm branch f32": norm(y=lambda t: t(2, 6, 64, dtype=F32)), "norm width 60": norm(x=lambda t: t(1, 2, 60), y=lambda t: t(1, 2, 60)),
    "norm no width": norm(x=lambda t: t(1, 2, 0), y=lambda t: t(1, 2, 0)), "norm too wide": norm(x=lambda t: t(1, 2, 8200), y=lambda t: t(1, 2, 8200)),
    "norm weight size": norm(w=lambda t: t(32)), "norm weight 2-D": norm(wb=lambda t: t(1, 64)), "norm weight f16": norm(w=lambda t: t(64, dtype=HF)),
    "norm scale alone": norm(shift=none), "norm shift alone": norm(scale=none), "norm table rows": norm(gate=lambda t: t(2, 64)),
    "norm table width": norm(scale=lambda t: t(3, 32)), "norm table f32": norm(shift=lambda t: t(3, 64, dtype=F32)), "norm no table rows": norm(
        gate=lambda t: t(0, 64), scale=none, shift=none), "norm no indices": norm(idx=none), "norm indices size": norm(idx=lambda t: t(5, dtype=I64)),
    "norm indices int32": norm(idx=lambda t: t(6, dtype=I32)), "norm branch kind": norm(bn=2), "norm kind": norm(kind=-1), "norm kind one plus": norm(kind=0x101),
    "norm weight without norm": norm(bn=-1), "norm scale inf": norm(a=float("inf")), "norm scale nan": norm(a=float("nan")), "norm scale f64": norm(a=1e39),
    "norm eps 0": norm(eps=0.0), "norm eps 1": norm(eps=1.0), "norm out f16": norm(out=HF),
    "route 1-D": route(x=lambda t: t(16, dtype=F32)), "route f64": route(x=lambda t: t(7, 16, dtype=torch.float64)), "route no experts": route(x=lambda t: t(7, 0, dtype=F32), k=1),
    "route too many": route(x=lambda t: t(2, 513, dtype=F32), local=513), "route k 0": route(k=0), "route k": route(k=17), "route k most": route(x=lambda t: t(2, 64, dtype=F32), k=33, local=64),
    "route bias size": route(bias=lambda t: t(15, dtype=F32)), "route bias bf16": route(bias=lambda t: t(16)), "route scoring": route(scoring=2),
    "route first": route(first=-1), "route local": route(first=1), "route no local": route(local=0), "route local all": route(local=17),
    "grouped dtypes": grouped(w=lambda t: t(3, 48, 32, dtype=I8)), "grouped bf16": grouped(a=lambda t: t(5, 32), w=lambda t: t(3, 48, 32)),
    "grouped 2-D": grouped(w=lambda t: t(48, 32, dtype=F8)), "grouped K": grouped(w=lambda t: t(3, 48, 48, dtype=F8)), "grouped K 24": grouped(
        a=lambda t: t(5, 24, dtype=F8), w=lambda t: t(3, 48, 24, dtype=F8)), "grouped N 40": grouped(w=lambda t: t(3, 40, 32, dtype=F8), sw=lambda t: t(3, 40, dtype=F32)),
    "grouped no groups": grouped(w=lambda t: t(0, 48, 32, dtype=F8)), "grouped too many": grouped(w=lambda t: t(513, 16, 32, dtype=F8), sw=lambda t: t(513, dtype=F32), ends=lambda t: t(513, dtype=I32)),
    "grouped scale": grouped(sa=lambda t: t(4, dtype=F32)), "grouped scale f16": grouped(sa=lambda t: t(5, dtype=HF)), "grouped w scale": grouped(sw=lambda t: t(144, dtype=F32)),
    "grouped w scale f64": grouped(sw=lambda t: t(3, 48, dtype=torch.float64)), "grouped ends": grouped(ends=lambda t: t(4, dtype=I32)), "grouped ends int64": grouped(ends=lambda t: t(3, dtype=I64)),
    "grouped rows int64": grouped(rows=lambda t: t(5, dtype=I64)), "grouped rows 2-D": grouped(rows=lambda t: t(5, 1, dtype=I32)), "grouped bias": grouped(bias=lambda t: t(48)),
    "grouped bias int8": grouped(bias=lambda t: t(3, 48, dtype=I8)), "grouped out": grouped(out=F32), "grouped act": grouped(act=2),
    "grouped exact int8": grouped(a=lambda t: t(5, 32, dtype=I8), w=lambda t: t(3, 48, 32, dtype=I8), exact=True),
    "combine 3-D": combine(y=lambda t: t(1, 12, 64)), "combine f32": combine(y=lambda t: t(12, 64, dtype=F32)), "combine width": combine(y=lambda t: t(12, 60)),
    "combine weights": combine(w=lambda t: t(6, 3, dtype=F32)), "combine weights bf16": combine(w=lambda t: t(6, 2)), "combine slots int64": combine(s=lambda t: t(6, 2, dtype=I64)),
    "combine no choices": combine(w=lambda t: t(6, 0, dtype=F32), s=lambda t: t(6, 0, dtype=I32)), "combine residual": combine(res=lambda t: t(5, 64)),
    "combine residual f16": combine(res=lambda t: t(6, 64, dtype=HF)), "combine gate alone": combine(gate=lambda t: t(4, 64), idx=lambda t: t(6, dtype=I64)),
    "combine gate f16": combine(res=lambda t: t(6, 64), gate=lambda t: t(4, 64, dtype=HF), idx=lambda t: t(6, dtype=I64)),
    "combine no indices": combine(res=lambda t: t(6, 64), gate=lambda t: t(4, 64)), "combine indices": combine(
        res=lambda t: t(6, 64), gate=lambda t: t(4, 64), idx=lambda t: t(4, dtype=I64)),
}


def outcome(call, device):
    try:
        out = call(Make(device))
    except RuntimeError as error:
        return "refused", str(error).splitlines()[0]
    return "accepted", [(tuple(o.shape), o.stride(), o.dtype) for o in (out if isinstance(out, (tuple, list)) else (out,))]


@pytest.mark.parametrize("name", sorted(ACCEPTED))
def test_accepted(name):
    kind, got = outcome(ACCEPTED[name], "meta")
    assert kind == "accepted", got


@pytest.mark.parametrize("name", sorted(REFUSED))
def test_refused(name):
    kind, got = outcome(REFUSED[name], "meta")
    assert kind == "refused" and got.startswith({"norm": "residual_norm", "route": "route", "grouped": "grouped_matmul",
                                                 "combine": "expert_combine"}[name.split()[0]]), got


def test_wrappers_refuse():
    t = Make("meta")
    x = t(2, 6, 64)
    grad = torch.zeros((2, 6, 64), dtype=BF, device="meta", requires_grad=True)
    with pytest.raises(ValueError, match="inference-only"):
        residual_norm(grad, x)
    with pytest.raises(ValueError, match="norm must be"):
        residual_norm(x, x, norm="group")
    with pytest.raises(ValueError, match="norm must be"):
        residual_norm(x, x, branch_norm="none")
    assert residual_norm(x, x)[1].shape == x.shape and len(residual_norm(x, x, out_dtype=F8)) == 3
    with pytest.raises(ValueError, match="inference-only"):
        ex.route(grad[0], 2)
    with pytest.raises(ValueError, match="scoring"):
        ex.route(t(3, 4), 2, scoring="relu")
    assert ex.route(t(3, 8), 2, first_expert=5).ends.shape == (3,)
    args = (t(5, 32, dtype=I8), t(5, dtype=F32), t(3, 48, 32, dtype=I8), t(3, 48, dtype=F32), t(3, dtype=I32))
    assert ex.grouped_matmul(*args).shape == (5, 48)  # int8: exact by itself
    with pytest.raises(ValueError, match="accumulation"):
        ex.grouped_matmul(*args, accumulation="fast")
    with pytest.raises(ValueError, match="activation"):
        ex.grouped_matmul(*args, activation="relu")
    y, w, s = t(12, 64), t(6, 2, dtype=F32), t(6, 2, dtype=I32)
    assert ex.combine(y, w, s, residual=t(2, 3, 64)).shape == (2, 3, 64)
    with pytest.raises(ValueError, match="indices"):
        ex.combine(y, w, s, residual=t(2, 3, 64), gate_table=t(4, 64), indices=t(2, dtype=I64))
    with pytest.raises(ValueError, match="residual"):
        ex.combine(y, w, s, residual=t(384))
    with pytest.raises(ValueError, match="inference-only"):
        ex.combine(y, w, s, residual=grad)


def test_module_refuses():
    up, down = torch.zeros(4, 64, 32, dtype=BF), torch.zeros(4, 32, 32, dtype=BF)
    for kw, match in ((dict(dtype="fp4"), "dtype"), (dict(activation="relu"), "activation"), (dict(scoring="max"), "scoring"),
                      (dict(accumulation="fast"), "accumulation"), (dict(activation="gelu_tanh"), "required"),
                      (dict(up_bias=torch.zeros(64)), "biases"), (dict(first_expert=-1), "experts"), (dict(total_experts=3), "experts")):
        with pytest.raises(ValueError, match=match):
            ex.W8A8Experts(up, down, 2, **kw)
    with pytest.raises(ValueError, match="experts"):
        ex.W8A8Experts(up, down, 5)
    with pytest.raises(ValueError, match="divisible"):
        ex.W8A8Experts(torch.zeros(4, 48, 40, dtype=BF), torch.zeros(4, 40, 24, dtype=BF), 2)


def test_features_and_library_paths():
    for feature in ("residual_norm", "experts"):
        assert runtime.Kernels.SPECS[feature] is not None
        d = runtime.Diagnostics()
        assert runtime.Kernels(d).get(feature, torch.zeros(1)) is None and len(d.fallbacks) == 1
    assert ex.library_path().name == "libxgen_amd.so"


def call(fn, good, **changes):
    names = list(good)
    assert set(changes) <= set(names)
    return lambda L: getattr(L, fn)(*({**good, **changes}[n] for n in names))


NORM = dict(x=16, xsb=0, xss=64, y=16, ysb=0, yss=64, batch=1, seq=4, width=64, bn=1, wb=16, kind=1, w=16, wdt=N.DTYPE_BF16, a=1.0, eps=1e-6,
            gate=16, gs=64, scale=16, ss=64, shift=16, ts=64, rows=3, idx=16, stream=16, out_dt=N.DTYPE_E4M3, out=16, tok=16, s=None)
ROUTE = dict(dt=N.DTYPE_F32, x=16, ld=16, tokens=300, experts=16, k=2, bias=None, scoring=0, ren=1, first=0, local=16, w=16, c=16, e=16, r=16,
             sl=16, ws=16, wsb=1 << 20, s=None)
GROUPED = dict(dt=N.DTYPE_E4M3, exact=0, a=16, lda=32, ar=5, w=16, ldw=32, wg=1536, M=5, N=48, K=32, G=3, ends=16, rows=None, sa=16, sas=1, sw=16,
               sws=1, bias=None, bdt=N.DTYPE_NONE, act=0, out=16, odt=N.DTYPE_BF16, ldo=48, s=None)
COMBINE = dict(dt=N.DTYPE_BF16, y=16, ldy=64, yr=12, w=16, sl=16, tokens=6, k=2, width=64, res=16, ldr=64, gate=16, gs=64, gr=4, idx=16, seq=3, out=16,
               s=None)
BAD, NO = N.ERR_INVALID_ARGUMENT, N.ERR_UNSUPPORTED


@pytest.mark.parametrize("fn,good,changes,status,needle", [
    ("xgen_residual_norm", NORM, dict(bn=2), BAD, b"branch norm kind"), ("xgen_residual_norm", NORM, dict(kind=0x101), BAD, b"norm kind"),
    ("xgen_residual_norm", NORM, dict(kind=-1), BAD, b"norm kind"), ("xgen_residual_norm", NORM, dict(out_dt=N.DTYPE_F16), BAD, b"output dtype"),
    ("xgen_residual_norm", NORM, dict(wdt=N.DTYPE_F16), BAD, b"weight dtype"), ("xgen_residual_norm", NORM, dict(w=None, wb=None), BAD, b"disagree"),
    ("xgen_residual_norm", NORM, dict(bn=-1), BAD, b"needs a branch norm"), ("xgen_residual_norm", NORM, dict(width=-8), BAD, b"bad shape"),
    ("xgen_residual_norm", NORM, dict(rows=0), BAD, b"bad shape"), ("xgen_residual_norm", NORM, dict(eps=0.0), BAD, b"eps"),
    ("xgen_residual_norm", NORM, dict(a=float("nan")), BAD, b"finite"), ("xgen_residual_norm", NORM, dict(xss=56), BAD, b"strides"),
    ("xgen_residual_norm", NORM, dict(gs=56), BAD, b"strides"), ("xgen_residual_norm", NORM, dict(shift=None), BAD, b"together"),
    ("xgen_residual_norm", NORM, dict(width=8200, xss=8200, yss=8200, gs=8200, ss=8200, ts=8200), NO, b"exceeds"),
    ("xgen_residual_norm", NORM, dict(batch=1 << 40, seq=1 << 40), NO, b"too many"), ("xgen_residual_norm", NORM, dict(y=None), BAD, b"null"),
    ("xgen_residual_norm", NORM, dict(idx=None), BAD, b"null"), ("xgen_residual_norm", NORM, dict(tok=None), BAD, b"null"),
    ("xgen_residual_norm", NORM, dict(x=24), NO, b"aligned"), ("xgen_residual_norm", NORM, dict(width=60), NO, b"multiples of 8"),
    ("xgen_route", ROUTE, dict(dt=N.DTYPE_I8), BAD, b"dtype"), ("xgen_route", ROUTE, dict(scoring=2), BAD, b"scoring"),
    ("xgen_route", ROUTE, dict(tokens=0), BAD, b"bad shape"), ("xgen_route", ROUTE, dict(k=17), BAD, b"bad shape"), ("xgen_route", ROUTE, dict(ld=15), BAD, b"bad shape"),
    ("xgen_route", ROUTE, dict(experts=513, ld=513), NO, b"experts"), ("xgen_route", ROUTE, dict(experts=64, ld=64, k=33), NO, b"choices"),
    ("xgen_route", ROUTE, dict(first=1), BAD, b"not among"), ("xgen_route", ROUTE, dict(local=0), BAD, b"not among"), ("xgen_route", ROUTE, dict(sl=None), BAD, b"null"),
    ("xgen_route", ROUTE, dict(tokens=1 << 30, k=2), NO, b"2^31"), ("xgen_route", ROUTE, dict(wsb=64), BAD, b"workspace"), ("xgen_route", ROUTE, dict(ws=None), BAD, b"workspace"),
    ("xgen_grouped_matmul", GROUPED, dict(dt=N.DTYPE_BF16), BAD, b"operand dtype"), ("xgen_grouped_matmul", GROUPED, dict(dt=N.DTYPE_I8, exact=1), BAD, b"exact"),
    ("xgen_grouped_matmul", GROUPED, dict(G=0), BAD, b"bad shape"), ("xgen_grouped_matmul", GROUPED, dict(ar=6), BAD, b"M rows"),
    ("xgen_grouped_matmul", GROUPED, dict(lda=16), BAD, b"leading"), ("xgen_grouped_matmul", GROUPED, dict(sas=2), BAD, b"activation scale"),
    ("xgen_grouped_matmul", GROUPED, dict(sws=48), BAD, b"weight scale"), ("xgen_grouped_matmul", GROUPED, dict(bias=16), BAD, b"bias dtype"),
    ("xgen_grouped_matmul", GROUPED, dict(act=3), BAD, b"activation"), ("xgen_grouped_matmul", GROUPED, dict(odt=N.DTYPE_F32), BAD, b"output dtype"),
    ("xgen_grouped_matmul", GROUPED, dict(G=513), NO, b"groups"), ("xgen_grouped_matmul", GROUPED, dict(ends=None), BAD, b"null"),
    ("xgen_grouped_matmul", GROUPED, dict(K=24, lda=32), NO, b"multiples of 16"), ("xgen_grouped_matmul", GROUPED, dict(lda=40), NO, b"aligned"),
    ("xgen_grouped_matmul", GROUPED, dict(w=24), NO, b"aligned"), ("xgen_grouped_matmul", GROUPED, dict(ldo=52), NO, b"aligned"),
    ("xgen_grouped_matmul", GROUPED, dict(N=1 << 20, K=1 << 12, lda=1 << 12, ldw=1 << 12, ldo=1 << 20), NO, b"2 GiB"),
    ("xgen_grouped_matmul", GROUPED, dict(lda=1 << 23), NO, b"32-bit"), ("xgen_grouped_matmul", GROUPED, dict(ldo=1 << 22), NO, b"32-bit"),
    ("xgen_grouped_matmul", GROUPED, dict(rows=16, ar=1 << 27), NO, b"indexed"),
    ("xgen_expert_combine", COMBINE, dict(dt=N.DTYPE_F32), BAD, b"dtype"), ("xgen_expert_combine", COMBINE, dict(k=0), BAD, b"bad shape"),
    ("xgen_expert_combine", COMBINE, dict(ldy=56), BAD, b"strides"), ("xgen_expert_combine", COMBINE, dict(res=None), BAD, b"gate"),
    ("xgen_expert_combine", COMBINE, dict(seq=4), BAD, b"gate"), ("xgen_expert_combine", COMBINE, dict(gr=0), BAD, b"gate"), ("xgen_expert_combine", COMBINE, dict(sl=None), BAD, b"null"),
    ("xgen_expert_combine", COMBINE, dict(idx=None), BAD, b"null"), ("xgen_expert_combine", COMBINE, dict(width=60), NO, b"multiples of 8"),
    ("xgen_expert_combine", COMBINE, dict(out=24), NO, b"aligned"), ("xgen_expert_combine", COMBINE, dict(tokens=3 << 30), NO, b"too many"),
])
def test_c_entry_checks(built_library, fn, good, changes, status, needle):
    L = N.lib()
    assert call(fn, good, **changes)(L) == status, L.xgen_last_error()
    assert needle in L.xgen_last_error()


def test_c_entries_without_work(built_library):
    L = N.lib()
    nulls = dict(x=None, y=None, gate=None, scale=None, shift=None, idx=None, stream=None, out=None, tok=None, w=None, wb=None, wdt=N.DTYPE_NONE)
    assert call("xgen_residual_norm", NORM, seq=0, **nulls)(L) == N.OK
    assert call("xgen_grouped_matmul", GROUPED, M=0, ar=0, a=None, w=None, ends=None, sa=None, sw=None, out=None)(L) == N.OK
    assert call("xgen_expert_combine", COMBINE, tokens=0, y=None, w=None, sl=None, out=None, idx=None)(L) == N.OK
    for experts, tokens in ((8, 32), (64, 32), (65, 16), (256, 8), (512, 4)):  # one launch up to there
        assert L.xgen_route_workspace_bytes(tokens, experts, 16) == 0
        assert L.xgen_route_workspace_bytes(tokens + 1, experts, 16) == -(-(tokens + 1) // 16) * 16 * 4
    assert L.xgen_route_workspace_bytes(4096, 8, 8) == 256 * 32 and L.xgen_route_workspace_bytes(4097, 8, 8) == 65 * 32
    assert L.xgen_route_workspace_bytes(32768, 8, 8) == 512 * 32 and L.xgen_route_workspace_bytes(32769, 8, 8) == 257 * 32
