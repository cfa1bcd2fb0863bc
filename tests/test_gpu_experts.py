"""The operators of a block with experts run together, as they would be used: against the same block
expert by expert on the package's ungrouped operators and against plain 64-bit products, captured in graphs,
on other streams, and by two ranks' shares.

Tolerance of W8A8Experts against 64 bits: with e4m3 operands both of a product's factors are off by at most 2^-4 of
their values (int8: half a unit of a row's largest / 127), so its relative 2-norm error is far below
the sum of both for independent errors; 0.08 (int8 0.03) holds with room for two products and the
activation.  The exact comparison is with the ungrouped operators."""
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import xgen_amd  # noqa: F401
from conftest import library_without
from xgen_amd import _native as N
from xgen_amd.operator.experts import W8A8Experts, combine, route
from xgen_amd.operator.residual_norm import residual_norm
from xgen_amd.operator.runtime import Diagnostics, Kernels

pytestmark = pytest.mark.gpu
xops = torch.ops.xgen_amd
FP8 = torch.float8_e4m3fn


def bits(t):
    return t.view(torch.uint8) if t.element_size() == 1 else t.view(torch.int16 if t.element_size() == 2 else torch.int32)


def same(a, b):
    return all(torch.equal(bits(x), bits(y)) for x, y in zip(a, b))


class Block:
    """norm behind a branch, gated residual and norm in front; router; experts; gated residual."""

    def __init__(self, cuda, seed, d=256, F=192, E=8, k=3, T=5, dtype="fp8", activation="swiglu", accumulation="mfma",
                 biases=True, **kw):
        g = torch.Generator(device=cuda).manual_seed(seed)
        self.g, self.d, self.E, self.cuda, self.dtype = g, d, E, cuda, dtype
        wide = 2 * F if activation == "swiglu" else F
        self.up = (torch.randn((E, wide, d), generator=g, device=cuda) * d ** -0.5).bfloat16()
        self.down = (torch.randn((E, d, F), generator=g, device=cuda) * F ** -0.5).bfloat16()
        self.up_bias = (torch.randn((E, wide), generator=g, device=cuda) * 0.1).bfloat16() if biases else None
        self.down_bias = (torch.randn((E, d), generator=g, device=cuda) * 0.1).bfloat16() if biases else None
        self.router = torch.randn((E, d), generator=g, device=cuda) * d ** -0.5
        self.experts = W8A8Experts(self.up, self.down, k, up_bias=self.up_bias, down_bias=self.down_bias, dtype=dtype,
                                   activation=activation, accumulation=accumulation, **kw)
        self.tables = (torch.randn((T, 4 * d), generator=g, device=cuda) * 0.3).bfloat16().chunk(4, dim=-1)
        self.weights = (1 + 0.1 * torch.randn((2, d), generator=g, device=cuda)).bfloat16()

    def inputs(self, B, S):
        x = torch.randn((B, S, self.d), generator=self.g, device=self.cuda).bfloat16()
        y = torch.randn((B, S, self.d), generator=self.g, device=self.cuda).bfloat16()
        return x, y, torch.randint(5, (S,), generator=self.g, device=self.cuda)

    def __call__(self, x, y, idx):
        gate, scale, shift, gate2 = self.tables
        stream, h = residual_norm(x, y, branch_weight=self.weights[0], weight=self.weights[1], gate_table=gate, scale=scale,
                                  shift=shift, indices=idx)
        logits = h.float() @ self.router.t()
        out = self.experts(h, logits, residual=stream, gate_table=gate2, indices=idx)
        return stream, h, logits, out


def expert_by_expert(block, h, logits, residual, gate, idx):
    """The module's arithmetic on the ungrouped operators, one expert at a time, summed by combine."""
    m = block.experts
    B, S, d = h.shape
    q, s = xops.quantize_rows(h.reshape(-1, d), m.dtype)
    plan = route(logits.reshape(-1, block.E), m.k, scoring=m.scoring, renormalize=m.renormalize)
    y = torch.zeros((B * S * m.k, d), dtype=torch.bfloat16, device=h.device)
    begin, exact = 0, m.accumulation == "exact" and m.dtype == FP8
    for e, end in enumerate(plan.ends.tolist()):
        if end > begin:
            r = plan.rows[begin:end].long()
            a = q.view(torch.uint8)[r].view(q.dtype)
            u, _ = xops.scaled_mm(a, m.up_weight[e], s[r], m.up_scale[e], None if m.up_bias is None else m.up_bias[e],
                                  torch.bfloat16, 0, False, exact)
            if m.activation == "swiglu":
                hq, hs, _ = xops.swiglu_quant(u[None], m.gate_first, m.dtype, 1, False)
            else:
                hq, hs = xops.quantize_rows(u, m.dtype, 1)
            y[begin:end], _ = xops.scaled_mm(hq, m.down_weight[e], hs, m.down_scale[e],
                                             None if m.down_bias is None else m.down_bias[e], torch.bfloat16, 0, False, exact)
        begin = end
    return combine(y, plan.weights, plan.slots, residual=residual, gate_table=gate, indices=idx)


@pytest.mark.parametrize("dtype,accumulation", [("fp8", "mfma"), ("fp8", "exact"), ("int8", "exact")])
@pytest.mark.parametrize("activation", ["swiglu", "gelu_tanh"])
@pytest.mark.parametrize("B,S", [(1, 1), (2, 37), (1, 700)])
def test_block_is_the_ungrouped_operators(cuda, dtype, accumulation, activation, B, S):
    block = Block(cuda, S, dtype=dtype, accumulation=accumulation, activation=activation, gate_first=S == 37)
    x, y, idx = block.inputs(B, S)
    stream, h, logits, out = block(x, y, idx)
    assert out.shape == x.shape
    assert torch.equal(bits(out), bits(expert_by_expert(block, h, logits, stream, block.tables[3], idx)))


@pytest.mark.parametrize("dtype,limit", [("fp8", 0.08), ("int8", 0.03)])
@pytest.mark.parametrize("activation", ["swiglu", "gelu_tanh"])
def test_experts_against_64_bits(cuda, dtype, limit, activation):
    block = Block(cuda, 3, dtype=dtype, activation=activation, scoring="sigmoid", renormalize=False)
    h = torch.randn((1, 333, block.d), generator=block.g, device=cuda).bfloat16()
    logits = torch.randn((1, 333, block.E), generator=block.g, device=cuda)
    logits[0, 5] = float("-inf")  # a padding row
    out = block.experts(h, logits)[0].double()
    x, p = h[0].double(), torch.sigmoid(logits[0].double())
    order = torch.sort(logits[0], dim=1, descending=True, stable=True).indices[:, :3]
    mask = torch.zeros_like(p).scatter_(1, order, 1.0) * torch.isfinite(logits[0])
    ref = torch.zeros_like(out)
    for e in range(block.E):
        u = x @ block.up[e].double().t() + block.up_bias[e].double()
        if activation == "swiglu":
            a, b = u.chunk(2, dim=1)
            u = a * torch.nn.functional.silu(b)
        else:
            u = torch.nn.functional.gelu(u, approximate="tanh")
        ref += (p * mask)[:, e:e + 1] * (u @ block.down[e].double().t() + block.down_bias[e].double())
    assert not out[5].any()
    assert ((out - ref).norm() / ref.norm()).item() <= limit


def test_quantized_rows_are_shared(cuda):
    """residual_norm's own fp8 rows through forward_quantized."""
    block = Block(cuda, 4)
    x, y, idx = block.inputs(2, 50)
    stream, q, s = residual_norm(x, y, weight=block.weights[1], out_dtype=FP8)
    logits = torch.randn((2, 50, block.E), generator=block.g, device=cuda)
    out = block.experts.forward_quantized(q, s, logits, x.shape, residual=stream)
    plan = route(logits.reshape(-1, block.E), 3)
    m = block.experts
    u = xops.grouped_matmul(q, s, m.up_weight, m.up_scale, plan.ends, plan.rows, m.up_bias, torch.bfloat16, 0, False)
    hq, hs, _ = xops.swiglu_quant(u[None], False, FP8, 1, False)
    v = xops.grouped_matmul(hq, hs, m.down_weight, m.down_scale, plan.ends, None, m.down_bias, torch.bfloat16, 0, False)
    assert torch.equal(out, combine(v, plan.weights, plan.slots, residual=stream))
    assert out.shape == x.shape


def test_ranks_shares_add_up(cuda):
    """Two ranks with half of the experts each: their sums are the whole one's, each rounded once (2^-8 of a share)."""
    block = Block(cuda, 5, biases=False, accumulation="exact")
    h = torch.randn((200, block.d), generator=block.g, device=cuda).bfloat16()
    logits = torch.randn((200, block.E), generator=block.g, device=cuda)
    logits[7, :4] = float("-inf")
    whole = block.experts(h, logits).double()
    shares = []
    for first in (0, 4):
        part = W8A8Experts(block.up[first:first + 4], block.down[first:first + 4], 3, accumulation="exact",
                           first_expert=first, total_experts=8)
        shares.append(part(h, logits).double())
    tol = 2.0 ** -8 * (shares[0].abs() + shares[1].abs() + whole.abs()) + 8 * 2.0 ** -24 * (shares[0].abs() + shares[1].abs())
    assert ((shares[0] + shares[1] - whole).abs() <= tol).all()
    assert not shares[0][7].any()


@pytest.mark.parametrize("B,S", [(1, 3), (1, 300), (2, 500)])
def test_captured_block_replays(cuda, B, S):
    """The whole chain in one graph, replayed on new inputs with eager work in between; two graphs of other sizes
    captured, replayed in turn."""
    block = Block(cuda, 6)
    graphs = []
    for seq in (S, S + 64):
        x, y, idx = block.inputs(B, seq)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(x, y, idx)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = block(x, y, idx)
        graphs.append((graph, x, y, idx, out))
    for rep in range(3):
        for graph, x, y, idx, out in graphs:
            new = block.inputs(*x.shape[:2])
            for old, n in zip((x, y, idx), new):
                old.copy_(n)
            graph.replay()
            torch.cuda.synchronize()
            assert same(out, block(*new)), rep
            torch.cuda.synchronize()


def test_two_streams_at_once(cuda):
    blocks = [Block(cuda, s) for s in (7, 8)]
    given = [b.inputs(1, 900) for b in blocks]
    ref = [b(*i) for b, i in zip(blocks, given)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        got = []
        for st, b, i in zip(streams, blocks, given):
            with torch.cuda.stream(st):
                got.append([b(*i) for _ in range(3)][-1])
        torch.cuda.synchronize()
        assert all(same(g, r) for g, r in zip(got, ref))


def test_no_tokens(cuda):
    block = Block(cuda, 9)
    out = block.experts(torch.empty((0, block.d), dtype=torch.bfloat16, device=cuda), torch.empty((0, block.E), device=cuda))
    assert out.shape == (0, block.d)


def test_module_through_the_runtime(cuda):
    d = Diagnostics()
    x = torch.zeros(1, device=cuda)
    kernels = Kernels(d)
    assert kernels.get("experts", x).W8A8Experts is W8A8Experts
    assert kernels.get("residual_norm", x).residual_norm is residual_norm
    assert not d.fallbacks


def test_weights_on_the_cpu_stay_there(cuda):
    up, down = torch.randn(2, 32, 16).bfloat16(), torch.randn(2, 16, 16).bfloat16()
    m = W8A8Experts(up, down, 1)
    assert m.up_weight.device.type == "cpu" and m.up_scale.shape == (2, 32)
    on = m.to(cuda)
    other = W8A8Experts(up.to(cuda), down.to(cuda), 1)
    assert torch.equal(bits(on.up_weight), bits(other.up_weight)) and torch.equal(on.down_scale, other.down_scale)
    h, logits = torch.randn(5, 16, device=cuda).bfloat16(), torch.randn(5, 2, device=cuda)
    assert torch.equal(on(h, logits), other(h, logits))


OLDER = """
import sys
sys.path.insert(0, sys.argv[1])
import torch, xgen_amd
from xgen_amd.operator.experts import combine, grouped_matmul, route
from xgen_amd.operator.residual_norm import residual_norm
x = torch.ones(1, 2, 16, dtype=torch.bfloat16, device="cuda")
q, s = torch.ops.xgen_amd.quantize_rows(x[0], torch.int8)
assert q.min().item() == 127
plan = torch.zeros(2, 1, dtype=torch.int32, device="cuda")
for call in (lambda: residual_norm(x, x), lambda: route(x[0].float(), 2),
             lambda: grouped_matmul(q, s, q.reshape(1, 2, 16).repeat(1, 8, 1), s[:1], plan[:1, 0]),
             lambda: combine(x[0], torch.ones(2, 1, device="cuda"), plan)):
    try:
        call()
    except RuntimeError as error:
        print(str(error).splitlines()[0])
"""


def test_library_from_before_the_operators(cuda, tmp_path):
    """XGEN_AMD_LIBRARY names a library of this ABI version without the entry points: the other operators run on it, and
    each of these names what it lacks."""
    older = N.library_path()
    symbols = ("xgen_residual_norm", "xgen_route", "xgen_grouped_matmul", "xgen_expert_combine")
    for symbol in symbols:
        folder = tmp_path / symbol
        folder.mkdir()
        older = library_without(older, symbol, folder)
    proc = subprocess.run([sys.executable, "-c", OLDER, str(Path(__file__).resolve().parents[1])], check=True, timeout=100,
                          stdout=subprocess.PIPE, text=True, env={**os.environ, "XGEN_AMD_LIBRARY": str(older)})
    lines = proc.stdout.strip().splitlines()[-4:]
    assert len(lines) == 4 and all(symbol in line for symbol, line in zip(symbols, lines)), lines
