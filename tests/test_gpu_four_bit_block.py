"""The 4-bit path as a block runs it: norm, QKV projection in 4 bits, norms and rotation of queries and keys where the
projection left them, the head-parallel exchange's layout, out-projection in 4 bits with the gated residual; on streams of their
own, from two threads, and in captured graphs that are replayed among eager work."""
import threading

import pytest
import torch

import oracle.ref as R
import xgen_amd  # noqa: F401
from test_gpu_graph import bits, capture, same
from test_gpu_mxfp4 import check_gated, check_product
from test_gpu_qk_norm_rope import check
from xgen_amd.operator import phaa_layout
from xgen_amd.operator.mxfp4 import MXFP4Linear, dequantize_mxfp4, quantize_mxfp4
from xgen_amd.operator.qk_norm_rope import qk_norm_rope, rotary_frequencies, rotary_table
from xgen_amd.operator.residual_norm import residual_norm

pytestmark = pytest.mark.gpu
BF = torch.bfloat16
HEADS, DIM = 56, 128


class Block:
    def __init__(self, seed, cuda, width=512):
        g = torch.Generator().manual_seed(seed)

        def weight(n, k):
            return (torch.randn((n, k), generator=g) * 0.02).to(BF).to(cuda)
        self.width = width
        self.qkv = MXFP4Linear(weight(3 * HEADS * DIM, width), torch.zeros(3 * HEADS * DIM, dtype=BF, device=cuda))
        self.out = MXFP4Linear(weight(width, HEADS * DIM), weight(1, width)[0])
        self.qw, self.kw = ((1 + 0.1 * torch.randn(DIM, generator=g)).to(BF).to(cuda) for _ in range(2))
        # three axes over the first 96 of a head's 128 values
        self.f = torch.cat([rotary_frequencies(2 * n, device=cuda)[0] for n in (16, 16, 16)])
        self.axes = torch.arange(48, device=cuda, dtype=torch.int32) // 16
        self.gate = torch.randn((4, width), generator=g).to(BF).to(cuda)

    def __call__(self, x, y, places, indices):
        """x, y BF16 [1, S, width], places int64 [S, 3], indices int64 [S]."""
        s = x.shape[1]
        stream, h = residual_norm(x, y)
        qkv = self.qkv(h)
        q, k, v = (t.unflatten(-1, (HEADS, DIM)) for t in qkv.chunk(3, dim=-1))
        cos, sin = rotary_table(places, self.f, axes=self.axes)
        q, k = qk_norm_rope(q, k, cos, sin, q_weight=self.qw, k_weight=self.kw)
        sends = [torch.empty((7, 4, s, 1, 2, DIM), dtype=BF, device=x.device) for _ in range(3)]
        phaa_layout.pack_qkv(q, k, v, *sends)
        attention = v.reshape(1, s, HEADS * DIM)  # (stands in for the attention)
        codes, scales = quantize_mxfp4(attention)
        sent = dequantize_mxfp4(codes, scales)     # what a peer takes from the packed rows
        return stream, h, qkv, cos, sin, q, k, *sends, sent, self.out.forward_gate_residual(attention, stream, self.gate, indices)


def inputs(seed, cuda, s, width=512):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((1, s, width), generator=g).to(BF).to(cuda), torch.randn((1, s, width), generator=g).to(BF).to(cuda),
            torch.randint(0, 128, (s, 3), generator=g).to(cuda), torch.randint(0, 4, (s,), generator=g).to(cuda))


@pytest.mark.parametrize("s", [1, 17, 301])
def test_block(cuda, s):
    block, given = Block(s, cuda), inputs(s, cuda, s)
    stream, h, qkv, cos, sin, q, k, qs, ks, vs, sent, out = block(*given)
    n = 3 * HEADS * DIM
    weight = (block.qkv.weight, block.qkv.weight_scales)
    check_product(quantize_mxfp4(h[0], rounding="ceil"), weight, s, n, block.width, block.qkv.bias, got=qkv[0])
    qv, kv, v = (t.unflatten(-1, (HEADS, DIM)) for t in qkv.chunk(3, dim=-1))
    assert same(check(qv, kv, cos, sin, q_weight=block.qw, k_weight=block.kw), (q, k))
    for x, send in ((q, qs), (k, ks), (v, vs)):
        assert torch.equal(send.cpu(), R.phaa_pack_qkv(x.cpu()))
    attention = v.reshape(s, HEADS * DIM)
    assert torch.equal(sent[0], dequantize_mxfp4(*quantize_mxfp4(attention)))
    check_gated(quantize_mxfp4(attention, rounding="ceil"), (block.out.weight, block.out.weight_scales), s, block.width, HEADS * DIM,
                block.out.bias, stream[0], block.gate, given[3], out[0])


def test_replays(cuda):
    """Captured once, replayed with new inputs and the program's own eager work between; two graphs alive at once."""
    block = Block(1, cuda)
    static = [list(inputs(1, cuda, s)) for s in (1, 130)]
    graphs = [capture(lambda given=given: block(*given)) for given in static]
    for rep in range(4):
        for given, (graph, out) in zip(static, graphs):
            for t, new in zip(given, inputs(20 + rep, cuda, given[0].shape[1])):
                t.copy_(new)
            graph.replay()
        torch.cuda.synchronize()
        for given, (graph, out) in zip(static, graphs):
            assert same(out, block(*given)), rep


def test_streams_and_threads(cuda):
    blocks = [Block(seed, cuda) for seed in (1, 2)]
    given = [inputs(seed, cuda, 200) for seed in (1, 2)]
    want = [b(*g) for b, g in zip(blocks, given)]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(4):
                got[i] = blocks[i](*given[i])
        stream.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for a, b in zip(got, want):
        assert all(torch.equal(bits(x), bits(y)) for x, y in zip(a, b))
