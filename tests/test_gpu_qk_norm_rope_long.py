"""qk_norm_rope on more tokens than one launch's threads: the bits of calls of its tokens alone."""
import pytest
import torch

import xgen_amd  # noqa: F401
from xgen_amd.operator.qk_norm_rope import qk_norm_rope, rotary_frequencies, rotary_table

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("heads,kv,tokens", [(1, 0, (1 << 26) + 77), (1, 1, (1 << 25) + 77)])
def test_tokens_past_one_launch(cuda, heads, kv, tokens):
    g = torch.Generator(device=cuda).manual_seed(tokens)
    q, k = (torch.empty((1, tokens, h, 8), dtype=BF, device=cuda) for h in (heads, kv))
    for t in (q, k):
        for first in range(0, tokens if t.numel() else 0, 1 << 22):
            last = min(tokens, first + (1 << 22))
            t[:, first:last] = torch.randn(t[:, first:last].shape, generator=g, device=cuda).to(BF)
    cos, sin = rotary_table(torch.arange(1000, device=cuda), rotary_frequencies(8, device=cuda)[0])
    at = torch.arange(tokens, device=cuda) % 1000
    got = qk_norm_rope(q, k, cos, sin, positions=at)
    for first in (0, (1 << 24) - 40, (1 << 25) - 40, tokens - 80):
        part = slice(first, first + 80)
        want = qk_norm_rope(q[:, part], k[:, part], cos, sin, positions=at[part])
        assert torch.equal(got[0][:, part], want[0]) and torch.equal(got[1][:, part], want[1]), first
    assert not any(torch.isnan(t).any() for t in got)
    norm = got[0].float().square().mean(-1)
    assert float(norm.min()) > 0.9  # (every head is written)
