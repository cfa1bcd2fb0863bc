"""A feed-forward of experts on the W8A8 path: router, ragged grouped products, weighted sum.

    route(logits, k)                        the k experts of each token, their weights, and the grouping of the
                                            (token, choice) pairs by expert
    grouped_matmul(q, scale, w, ws, ends)   one W8A8 product per group of rows, in one launch
    combine(y, weights, slots)              each token's weighted sum of its experts' rows, with the gated
                                            residual behind it
    W8A8Experts                             a module of the three, with the path's quantizers between them

Nothing is dropped and nothing waits for the host: a plan has tokens * k pairs, and the group ends stay on the
device.  Tokens whose logits are all -inf (padding) take no expert; with `first_expert` / `local_experts`
only those experts' pairs are in the plan (an expert-parallel rank's share: the ranks' sums add up).
grouped_matmul also serves other ragged groups with weights of their own, such as the text and video
rows of a dual-stream block (`ends` = the cumulated row counts).

Inference only: ValueError for tensors that require grad, RuntimeError for contract violations.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import nn

from .. import _native as N
from ..ops import xops
from .h3_fp8 import _ACCUMULATIONS, _ACTIVATIONS, _device_weight

# (the overloads themselves: half a microsecond less a call)
_route, _grouped_matmul, _combine = xops.route.default, xops.grouped_matmul.default, xops.expert_combine.default
_SCORINGS = {"softmax": N.ROUTE_SOFTMAX, "sigmoid": N.ROUTE_SIGMOID}
_FORMATS = {"fp8": torch.float8_e4m3fn, "int8": torch.int8}


def library_path():
    """The library holding the kernels (XGEN_AMD_LIBRARY overrides it)."""
    return N.library_path()


def _inference_only(*tensors):
    for t in tensors:
        if t is not None and t.requires_grad:
            raise ValueError("the expert operators are inference-only; detach parameters explicitly")


class Routing(NamedTuple):
    weights: torch.Tensor  # float32 [T, k]
    experts: torch.Tensor  # int32 [T, k], -1 where a token takes fewer than k
    ends: torch.Tensor     # int32 [local experts]: pairs up to each expert's last
    rows: torch.Tensor     # int32 [T * k]: token of each pair, -1 behind the last
    slots: torch.Tensor    # int32 [T, k]: place of each pair, -1 if no expert here takes it


def route(logits, k, *, bias=None, scoring="softmax", renormalize=True, first_expert=0, local_experts=None):
    """The k experts of largest logits + bias (ties to the lowest; -inf and NaN never), in that order, for logits
    BF16/F16/F32 [T, E].  Weights come from the logits without the bias: softmax over all experts, or sigmoid;
    `renormalize` divides them by their sum over the taken experts.  The plan groups the pairs of experts
    [first_expert, first_expert + local_experts) (default: all) in the order (expert, token, choice).

    `bias` is a prior on the logits, whatever the scoring.  A balancing bias that a router was trained with on its
    scores (softmax(logits) + b, sigmoid(logits) + b) ranks otherwise: such a router gives its biased scores as `logits`,
    takes the plan, and gathers its weights from the scores by `experts`."""
    _inference_only(logits, bias)
    if scoring not in _SCORINGS:
        raise ValueError(f"scoring must be one of {sorted(_SCORINGS)}")
    if local_experts is None:
        local_experts = logits.shape[-1] - first_expert
    return Routing(*_route(logits, k, bias, _SCORINGS[scoring], renormalize, first_expert, local_experts))


def grouped_matmul(q, scale, weight, weight_scale, ends, *, rows=None, bias=None, out_dtype=torch.bfloat16, activation=None,
                   accumulation="exact"):
    """[M, N]: row m, of group e where ends[e - 1] <= m < ends[e], is (q[r] . weight[e]^T) * (scale[r] *
    weight_scale[e]) + bias[e] with r = rows[m] (m itself without rows), rounded once, or its GELU-tanh.
    q e4m3fn / int8 [R, K] with scale float32 [R] (or one); weight of its dtype [G, N, K], weight_scale [G, N]
    or [G]; ends int32 [G] and rows int32 [M] as route gives them; bias [G, N].  Rows behind the last group
    are zeros; a row index outside q gives a NaN row.  `accumulation`: as H3FP8Linear's (int8 is exact)."""
    _inference_only(scale, weight_scale, bias)
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unsupported activation {activation!r}")
    if accumulation not in _ACCUMULATIONS:
        raise ValueError(f"accumulation must be one of {_ACCUMULATIONS}")
    return _grouped_matmul(q, scale, weight, weight_scale, ends, rows, bias, out_dtype, _ACTIVATIONS[activation],
                           accumulation == "exact" and q.dtype == torch.float8_e4m3fn)


def combine(y, weights, slots, *, residual=None, gate_table=None, indices=None):
    """sum_j weights[t, j] * y[slots[t, j]] in fp32, for y BF16/F16 [M, H] and a route's weights and slots; with
    a residual [T, H] or [B, S, H] (T = B * S), residual + gate_table[indices[s]] * that sum (gate 1 without a
    table).  Shaped as the residual, [T, H] without one.  A slot of -1 adds nothing."""
    _inference_only(y, weights, residual, gate_table)
    if residual is None or residual.dim() == 2:
        return _combine(y, weights, slots, residual, gate_table, indices)
    if residual.dim() != 3:
        raise ValueError("combine: residual [T, H] or [B, S, H] required")
    if gate_table is not None and (indices is None or indices.shape != (residual.shape[1],)):
        raise ValueError("combine: int64 indices [S] required with a gate table")
    out = _combine(y, weights, slots, residual.reshape(-1, residual.shape[2]), gate_table, indices)
    return out.reshape(residual.shape)


class W8A8Experts(nn.Module):
    """Experts with W8A8 projections: quantize each token once, route, up-project its row for its experts,
    activate and requantize in one pass, down-project, sum.

    up [E, 2F, d] with activation "swiglu" (rows [hidden | gate], [gate | hidden] with gate_first) or
    [E, F, d] with "gelu_tanh"; down [E, d, F]; biases [E, 2F or F] and [E, d].  Weights are quantized per
    output channel on construction, to `dtype` "fp8" or "int8", and stay on the device they came from.
    `accumulation` as H3FP8Linear's.  `total_experts` with `first_expert`: these are experts [first_expert,
    first_expert + E) of so many (expert parallelism); the output is their share of the sum.
    """

    def __init__(self, up, down, k, *, up_bias=None, down_bias=None, dtype="fp8", activation="swiglu", gate_first=False,
                 scoring="softmax", renormalize=True, accumulation="exact", first_expert=0, total_experts=None):
        super().__init__()
        if dtype not in _FORMATS:
            raise ValueError(f"dtype must be one of {sorted(_FORMATS)}")
        if activation not in ("swiglu", "gelu_tanh"):
            raise ValueError("activation must be 'swiglu' or 'gelu_tanh'")
        if scoring not in _SCORINGS:
            raise ValueError(f"scoring must be one of {sorted(_SCORINGS)}")
        if accumulation not in _ACCUMULATIONS:
            raise ValueError(f"accumulation must be one of {_ACCUMULATIONS}")
        if up.ndim != 3 or down.ndim != 3 or up.shape[0] != down.shape[0] or up.shape[2] != down.shape[1] \
                or up.shape[1] != down.shape[2] * (2 if activation == "swiglu" else 1):
            raise ValueError("up [E, 2F or F, d] and down [E, d, F] required")
        if any(n % 16 for n in (*up.shape[1:], *down.shape[1:])):
            raise ValueError("expert projection dimensions must be divisible by 16")
        for b, w in ((up_bias, up), (down_bias, down)):
            if b is not None and b.shape != w.shape[:2]:
                raise ValueError("biases must be [E, output features]")
        self.experts, self.in_features, self.hidden = up.shape[0], up.shape[2], down.shape[2]
        self.total_experts = first_expert + self.experts if total_experts is None else total_experts
        if first_expert < 0 or first_expert + self.experts > self.total_experts or not 0 < k <= self.total_experts:
            raise ValueError("k and [first_expert, first_expert + E) must lie among the experts")
        self.k, self.first_expert = k, first_expert
        self.dtype, self.activation, self.gate_first = _FORMATS[dtype], activation, gate_first
        self.scoring, self.renormalize, self.accumulation = scoring, renormalize, accumulation
        for name, value, bias in (("up", up, up_bias), ("down", down, down_bias)):
            packed, scale = xops.quantize_rows(_device_weight(value), self.dtype)
            self.register_buffer(f"{name}_weight", packed.to(value.device))
            self.register_buffer(f"{name}_scale", scale.reshape(value.shape[:2]).to(value.device))
            self.register_buffer(f"{name}_bias", bias.detach().clone() if bias is not None else None)

    def forward(self, x, logits, *, bias=None, residual=None, gate_table=None, indices=None):
        """x BF16 [..., d], logits [..., E] of the router (bias: route's, on the logits and not on their scores); the
        experts' sum shaped as x, or the gated residual behind it (combine's)."""
        if x.dtype != torch.bfloat16 or x.shape[-1] != self.in_features:
            raise ValueError(f"W8A8Experts requires a BF16 [..., {self.in_features}] input")
        _inference_only(x, logits)
        q, scale = xops.quantize_rows(x.reshape(-1, x.shape[-1]), self.dtype)
        return self.forward_quantized(q, scale, logits, x.shape, bias=bias, residual=residual, gate_table=gate_table,
                                      indices=indices)

    def forward_quantized(self, q, scale, logits, shape, *, bias=None, residual=None, gate_table=None, indices=None):
        """forward of rows that are quantized already (residual_norm's, nq2.norm_affine_quant's): q [T, d] and
        scale [T]; shape: of the result."""
        if logits.shape[-1] != self.total_experts:
            raise ValueError(f"logits of {self.total_experts} experts required")
        plan = route(logits.reshape(-1, logits.shape[-1]), self.k, bias=bias, scoring=self.scoring,
                     renormalize=self.renormalize, first_expert=self.first_expert, local_experts=self.experts)
        if plan.weights.shape[0] != q.shape[0]:
            raise ValueError("W8A8Experts: one row of logits per token required")
        u = grouped_matmul(q, scale, self.up_weight, self.up_scale, plan.ends, rows=plan.rows, bias=self.up_bias,
                           accumulation=self.accumulation)
        if self.activation == "swiglu":
            h, h_scale, _ = xops.swiglu_quant(u[None], self.gate_first, self.dtype, 1, False)
        else:
            h, h_scale = xops.quantize_rows(u, self.dtype, N.ACT_GELU_TANH)
        y = grouped_matmul(h, h_scale, self.down_weight, self.down_scale, plan.ends, bias=self.down_bias,
                           accumulation=self.accumulation)
        out = combine(y, plan.weights, plan.slots, residual=residual, gate_table=gate_table, indices=indices)
        return out if residual is not None else out.reshape(*shape[:-1], self.in_features)

    def extra_repr(self):
        return (f"experts={self.experts} of {self.total_experts} from {self.first_expert}, k={self.k}, d={self.in_features}, "
                f"hidden={self.hidden}, dtype={self.dtype}, activation={self.activation}, scoring={self.scoring}, "
                f"renormalize={self.renormalize}, accumulation={self.accumulation}")
