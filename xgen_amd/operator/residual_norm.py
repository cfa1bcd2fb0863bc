"""The norms behind and in front of a block's branch, with its gate and residual scale, in one kernel.

    stream = residual_scale * residual + gate_table[i] * (norm_b(branch) * branch_weight)
    rows   = norm(stream) * weight * (1 + scale[i]) + shift[i],   i = indices[position]

What a block that norms its branch's output (a "sandwich" norm) runs between two of its linears: the
end of one branch and the front end of the next, where gate_residual and then nq2.norm_affine_quant do it for a
block that norms in front only.  `branch_norm` "rms", "layer" or None (the branch as it is: the gated
residual), `norm` "rms" or "layer"; each weight, the gate and the scale / shift pair may be left out.
`out_dtype` bfloat16 returns (stream, rows), both BF16 [B, S, H]; float8_e4m3fn or int8 returns (stream,
q [B*S, H], token_scale float32 [B*S]), the rows quantized per token as runtime.quant_matmul takes them.

Arithmetic is fp32 from the loads to the stores: the stream and the rows are each rounded once (the front ends
of nq2 round after every eager bf16 operation, as their reference does).  An index outside the tables makes
its row NaN (quantized rows: a NaN scale).  Inference only: ValueError for a tensor that requires grad,
RuntimeError for contract violations.
"""
from __future__ import annotations

import torch

from .. import _native as N
from ..ops import xops

_residual_norm = xops.residual_norm.default  # (the overload itself: half a microsecond less a call)
_NORMS = {"rms": N.NORM_RMS, "layer": N.NORM_LAYER}


def library_path():
    """The library holding the kernel (XGEN_AMD_LIBRARY overrides it)."""
    return N.library_path()


def residual_norm(residual, branch, *, branch_weight=None, gate_table=None, residual_scale=1.0, weight=None, scale=None,
                  shift=None, indices=None, branch_norm="rms", norm="rms", eps=1e-6, out_dtype=torch.bfloat16):
    """residual, branch BF16 [B, S, H]; weights BF16/F32 [H]; tables BF16 [T, H]; indices int64 [S];
    eps in [2^-126, 1)."""
    if (residual.requires_grad or branch.requires_grad or (branch_weight is not None and branch_weight.requires_grad)
            or (weight is not None and weight.requires_grad) or (gate_table is not None and gate_table.requires_grad)
            or (scale is not None and scale.requires_grad) or (shift is not None and shift.requires_grad)):
        raise ValueError("residual_norm is inference-only; detach parameters explicitly")
    if norm not in _NORMS or (branch_norm is not None and branch_norm not in _NORMS):
        raise ValueError(f"norm must be one of {sorted(_NORMS)}, branch_norm one of them or None")
    stream, rows, token_scale = _residual_norm(
        residual, branch, branch_weight, weight, gate_table, scale, shift, indices,
        N.NORM_NONE if branch_norm is None else _NORMS[branch_norm], _NORMS[norm], float(residual_scale), float(eps),
        out_dtype)
    return (stream, rows) if out_dtype == torch.bfloat16 else (stream, rows, token_scale)
