"""Norms of queries and keys over each head with their position rotation in one kernel, and its table of angles.

What a block runs between its fused QKV projection and the attention (or phaa_layout.pack_qkv in front of a
head-parallel one): `qk_norm_rope` reads the heads where the projection left them.

    cos, sin = rotary_table(positions, frequencies, axes=...)   once per request, or per step for new positions
    q, k = qk_norm_rope(q, k, cos, sin, q_weight=..., k_weight=...)

Rotations: layout "half" turns the pairs (i, i + R/2), "interleaved" (2 i, 2 i + 1), of the first R values of a head,
R = 2 * cos.shape[1]; the rest of the head is normed only.  `rotary_frequencies` gives the frequencies, also scaled
for contexts longer than a model was trained on.

Inference only: ValueError for a tensor that requires grad, RuntimeError for contract violations.
"""
from __future__ import annotations

import math

import torch

from .. import _native as N
from ..ops import xops

_qk_norm_rope, _rotary_table = xops.qk_norm_rope.default, xops.rotary_table.default
_NORMS = {None: N.NORM_NONE, "rms": N.NORM_RMS, "layer": N.NORM_LAYER}
_LAYOUTS = ("half", "interleaved")


def library_path():
    """The library holding the kernels (XGEN_AMD_LIBRARY overrides it)."""
    return N.library_path()


def qk_norm_rope(q, k, cos, sin, *, positions=None, q_weight=None, k_weight=None, norm="rms", eps=1e-6, layout="half"):
    """(q', k') contiguous, of q [B, S, H, D] and k [B, S, Hk, D], BF16/F16 views with any strides (read in place where
    heads start on 16 bytes, copied otherwise); D a multiple of 8 up to 512.  `norm` "rms", "layer" (without a bias) or None over each
    head, with weights BF16/F16/F32 [D] or None.  cos, sin float32 [P, R/2]; positions int64 [S] or [B, S] into them, None
    for 0 .. S - 1; a position outside makes its token's heads NaN.  Arithmetic is fp32, rounded once."""
    if q.requires_grad or k.requires_grad or any(t is not None and t.requires_grad for t in (q_weight, k_weight, cos, sin)):
        raise ValueError("qk_norm_rope is inference-only; detach parameters explicitly")
    if norm not in _NORMS:
        raise ValueError("norm must be 'rms', 'layer' or None")
    if layout not in _LAYOUTS:
        raise ValueError(f"layout must be one of {_LAYOUTS}")
    return _qk_norm_rope(q, k, cos, sin, positions, q_weight, k_weight, _NORMS[norm], float(eps), layout == "interleaved")


def rotary_table(positions, frequencies, *, axes=None, factor=1.0):
    """(cos, sin) float32 [P, R/2] of positions int64 [P] or [P, A] (A axes, as time, height and width) and frequencies
    float64 [R/2]: factor * cos(positions[p, axes[i]] * frequencies[i]), the angle in 64 bits.  axes int32 [R/2]
    names each pair's axis (None: the first).  NaN for an axis outside and for angles from 2^36 on."""
    return _rotary_table(positions, frequencies, axes, float(factor))


def rotary_frequencies(dim, *, base=10000.0, scaling=None, factor=1.0, trained_length=None, low=1.0, high=32.0,
                       device=None):
    """(frequencies float64 [dim/2], table factor) of base^(-2 i / dim), scaled for contexts `factor` times as long:

      None       as they are
      "linear"   all divided by factor (positions interpolated)
      "base"     the base raised to base * factor^(dim / (dim - 2)): the slowest pair as "linear", the fastest as it is
                 (NTK-aware scaling)
      "bands"    by turns over trained_length, t = frequency * trained_length / (2 pi): pairs of `high` turns or more
                 as they are, of `low` or fewer divided by factor, between them blended in proportion to t
                 (configurations' rope type "llama3"; they give low_freq_factor and high_freq_factor, 1 and 4)
      "ramp"     as "bands", but blended in proportion to the pair's place between those of `high` and `low` turns,
                 and the table scaled by 0.1 ln(factor) + 1 (attention logits grow by its square)
                 (YaRN, with its whole-pair ends and its guard of 0.001; beta_fast is high, beta_slow low)
    """
    if dim <= 0 or dim % 2:
        raise ValueError("rotary_frequencies: an even dim required")
    if not (base > 1 and factor >= 1):
        raise ValueError("rotary_frequencies: base above 1 and factor of at least 1 required")
    at = torch.arange(dim // 2, dtype=torch.float64, device=device)
    if scaling == "base":
        if dim == 2:
            raise ValueError("rotary_frequencies: scaling 'base' needs dim above 2")
        base = base * factor ** (dim / (dim - 2))
    f = base ** (-2.0 * at / dim)
    if scaling in (None, "base"):
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    if scaling not in ("bands", "ramp"):
        raise ValueError("scaling must be None, 'linear', 'base', 'bands' or 'ramp'")
    if trained_length is None or not trained_length > 0 or not 0 < low < high:
        raise ValueError(f"rotary_frequencies: scaling {scaling!r} needs trained_length and 0 < low < high")
    if scaling == "bands":
        kept = ((f * trained_length / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
        return f * kept + f / factor * (1 - kept), 1.0

    def place(turns):  # of the pair that makes so many turns
        return dim * math.log(trained_length / (2 * math.pi * turns)) / (2 * math.log(base))

    first, last = max(math.floor(place(high)), 0), min(math.ceil(place(low)), dim - 1)
    kept = 1 - ((at - first) / max(last - first, 0.001)).clamp(0, 1)
    return f * kept + f / factor * (1 - kept), 0.1 * math.log(factor) + 1.0
