"""combine against its formula in 64 bits.  Tolerance: one rounding of half a step (bf16 2^-8, f16 2^-11; f16
subnormals 2^-25), and k + 3 fp32 operations in front of it, each off by 2^-24 of the magnitudes summed."""
import pytest
import torch

import xgen_amd  # noqa: F401
from xgen_amd.operator.experts import combine, route

pytestmark = pytest.mark.gpu


def check(cuda, y, w, slots, residual=None, gate_table=None, indices=None):
    out = combine(y, w, slots, residual=residual, gate_table=gate_table, indices=indices)
    T, k = w.shape
    parts = torch.where((slots >= 0)[..., None], y.double()[slots.long().clamp(min=0)] * w.double()[..., None], 0.0)
    ref, mag = parts.sum(1), parts.abs().sum(1)
    flat = None if residual is None else residual.reshape(T, -1).double()
    if gate_table is not None:
        g = gate_table.double()[indices].repeat(T // indices.shape[0], 1)
        ref, mag = ref * g, mag * g.abs()
    if flat is not None:
        ref, mag = ref + flat, mag + flat.abs()
    half = torch.finfo(y.dtype).eps / 2
    assert out.dtype == y.dtype and out.shape == (ref.shape if residual is None else residual.shape)
    tol = half * ref.abs() + (k + 3) * 2.0 ** -24 * mag * (1 + half) + (2.0 ** -25 if y.dtype == torch.float16 else 0)
    assert ((out.reshape(T, -1).double() - ref).abs() <= tol).all()
    return out


def inputs(cuda, T, k, H, seed, dtype=torch.bfloat16, E=16, padded=0):
    g = torch.Generator(device=cuda).manual_seed(seed)
    x = torch.randn((T, E), generator=g, device=cuda)
    x[T - padded:] = float("-inf")
    plan = route(x, k)
    return torch.randn((T * k, H), generator=g, device=cuda).to(dtype), plan.weights, plan.slots, g


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T,k,H", [(1, 1, 8), (1, 8, 2048), (3, 3, 520), (64, 2, 512), (65, 5, 504), (7, 16, 5376),
                                   (2000, 4, 1032), (9000, 6, 2048)])
def test_sizes(cuda, T, k, H, dtype):
    y, w, slots, g = inputs(cuda, T, k, H, T + H, dtype)
    check(cuda, y, w, slots)
    r = torch.randn((T, H), generator=g, device=cuda).to(dtype)
    check(cuda, y, w, slots, r)
    gate = torch.randn((5, 2 * H), generator=g, device=cuda).to(dtype)[:, H:]
    check(cuda, y, w, slots, r, gate, torch.randint(5, (T,), generator=g, device=cuda))


def test_batches_share_indices(cuda):
    B, S, k, H = 3, 50, 2, 256
    y, w, slots, g = inputs(cuda, B * S, k, H, 1)
    r = torch.randn((B, S, H), generator=g, device=cuda).bfloat16()
    gate = torch.randn((5, H), generator=g, device=cuda).bfloat16()
    check(cuda, y, w, slots, r, gate, torch.randint(5, (S,), generator=g, device=cuda))


def test_tokens_without_experts(cuda):
    y, w, slots, g = inputs(cuda, 40, 4, 64, 2, padded=7)
    r = torch.randn((40, 64), generator=g, device=cuda).bfloat16()
    assert not check(cuda, y, w, slots)[33:].any()
    assert torch.equal(check(cuda, y, w, slots, r)[33:], r[33:])
    # rows that no slot names, and the weights of absent slots, are not read into the sum
    y2, w2 = y.clone(), w.clone()
    y2[int(slots.max()) + 1:] = float("nan")
    w2[slots < 0] = float("nan")
    assert torch.equal(combine(y, w, slots), combine(y2, w2, slots))


def test_bad_slots_and_indices_make_their_row_nan(cuda):
    y, w, slots, g = inputs(cuda, 20, 3, 128, 3)
    r = torch.randn((20, 128), generator=g, device=cuda).bfloat16()
    gate = torch.randn((4, 128), generator=g, device=cuda).bfloat16()
    idx = torch.randint(4, (20,), generator=g, device=cuda)
    clean = combine(y, w, slots, residual=r, gate_table=gate, indices=idx)
    bad_slots, bad_idx = slots.clone(), idx.clone()
    bad_slots[4, 1], bad_slots[5, 0] = y.shape[0], 2 ** 31 - 1
    bad_idx[6], bad_idx[7], bad_idx[19] = 4, -1, -(1 << 40)
    got = combine(y, w, bad_slots, residual=r, gate_table=gate, indices=bad_idx)
    rows = torch.zeros(20, dtype=torch.bool, device=cuda)
    rows[[4, 5, 6, 7, 19]] = True
    assert torch.isnan(got[rows].float()).all() and torch.equal(got[~rows], clean[~rows])


def test_views(cuda):
    y, w, slots, g = inputs(cuda, 30, 2, 256, 4)
    wide = torch.zeros((60, 512), dtype=torch.bfloat16, device=cuda)
    wide[:, 256:] = y
    ref = combine(y, w, slots)
    assert torch.equal(combine(wide[:, 256:], w, slots), ref)
    assert torch.equal(combine(y, w.t().contiguous().t(), slots.t().contiguous().t(), residual=None), ref)
    r = torch.randn((60, 300), generator=g, device=cuda).bfloat16()[::2, 5:261]
    assert torch.equal(combine(y, w, slots, residual=r), combine(y, w, slots, residual=r.contiguous()))


def test_no_tokens(cuda):
    y = torch.empty((0, 64), dtype=torch.bfloat16, device=cuda)
    w, s = torch.empty((0, 2), device=cuda), torch.empty((0, 2), dtype=torch.int32, device=cuda)
    assert combine(y, w, s).shape == (0, 64)
    # no rows at all: every slot is absent
    w, s = torch.ones((3, 2), device=cuda), torch.full((3, 2), -1, dtype=torch.int32, device=cuda)
    assert not combine(y, w, s).any()


def test_rows_past_32_bit_offsets(cuda):
    """y of 5 GB: slots whose rows start past 2^32 bytes."""
    H, M = 8192, 310000
    y = torch.empty((M, H), dtype=torch.bfloat16, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(5)
    y[-64:] = torch.randn((64, H), generator=g, device=cuda).bfloat16()
    slots = torch.randint(M - 64, M, (16, 4), generator=g, device=cuda, dtype=torch.int32)
    w = torch.rand((16, 4), generator=g, device=cuda)
    got = combine(y, w, slots)
    assert torch.equal(got, combine(y[-64:], w, slots - (M - 64)))
