"""4-bit microscaled projections (MXFP4) beside the path's 8-bit ones, on the gfx950 matrix cores.

    quantize_mxfp4(x)                       rows as e2m1 codes with one power-of-two scale per 32 values
    dequantize_mxfp4(codes, scales)         the values they stand for
    mxfp4_matmul(codes, scales, w, ws)      their product, with bias, GELU-tanh or the gated residual behind it
    MXFP4Linear                             a projection with 4-bit weights and activations
    pack_scales / unpack_scales             scale bytes [rows, K / 32] to and from the layout the product reads

A code holds 0, 0.5, 1, 1.5, 2, 3, 4 or 6 with a sign, two codes a byte (the value of even k in the low four bits); a scale
is a byte e, 2^(e - 127).  That is the OCP microscaling format's MXFP4, so weights packed elsewhere are taken as
they are, but for the order of their scale bytes (`pack_scales`).  A product reads half the bytes of an 8-bit one
and runs at twice its rate on the matrix cores.

`rounding` chooses a block's scale from its largest |x|: "floor", the format's rule 2^(floor(log2 max) - 2),
where values above 6 scales (up to 8) saturate, or "ceil", the least power of two at which none does.

Inference only: ValueError for tensors that require grad, RuntimeError for contract violations.
"""
from __future__ import annotations

import torch
from torch import nn

from .. import _native as N
from ..ops import xops
from .h3_fp8 import _ACTIVATIONS, _device_weight

# (the overloads themselves: half a microsecond less a call)
_quantize, _dequantize, _matmul = xops.quantize_mxfp4.default, xops.dequantize_mxfp4.default, xops.mxfp4_matmul.default
_ROUNDINGS = {"floor": N.MX_FLOOR, "ceil": N.MX_CEIL}


def library_path():
    """The library holding the kernels (XGEN_AMD_LIBRARY overrides it)."""
    return N.library_path()


def _inference_only(*tensors):
    for t in tensors:
        if t is not None and t.requires_grad:
            raise ValueError("the MXFP4 operators are inference-only; detach parameters explicitly")


def _rounding(name):
    if name not in _ROUNDINGS:
        raise ValueError(f"rounding must be one of {sorted(_ROUNDINGS)}")
    return _ROUNDINGS[name]


def quantize_mxfp4(x, *, rounding="floor"):
    """(codes uint8 [..., K/2], scales uint8 [ceil(K/256), rows rounded up to even, 8]) of x BF16/F16 [..., K], K a
    multiple of 32.  Scales: eight bytes of a row's 256 values, block i of 32 at (i % 2) * 4 + i // 2.  A block with
    an inf or NaN is NaN (scale byte 255)."""
    _inference_only(x)
    return _quantize(x, _rounding(rounding))


def dequantize_mxfp4(codes, scales, *, dtype=torch.bfloat16):
    """The values of packed rows, [..., K] of dtype bfloat16 (exact for what quantize_mxfp4 gave), float32 (exact)
    or float16 (rounded)."""
    return _dequantize(codes, scales, dtype)


def pack_scales(scales):
    """Scale bytes [rows, K/32] (uint8, or float8_e8m0fnu as bytes) in the layout of quantize_mxfp4's."""
    if scales.dim() != 2 or scales.element_size() != 1:
        raise ValueError("pack_scales: one byte per 32 values, [rows, K/32], required")
    scales = scales.view(torch.uint8)
    rows, blocks = scales.shape
    out = scales.new_zeros((rows + rows % 2, (blocks + 7) // 8 * 8))
    out[:rows, :blocks] = scales
    return out.reshape(out.shape[0], -1, 4, 2).permute(1, 0, 3, 2).reshape(-1, out.shape[0], 8).contiguous()


def unpack_scales(scales, rows, K):
    """Scale bytes uint8 [rows, K/32] of quantize_mxfp4's layout for rows of K values."""
    if scales.dtype != torch.uint8 or K % 32 or tuple(scales.shape) != ((K + 255) // 256, rows + rows % 2, 8):
        raise ValueError("unpack_scales: scales uint8 [ceil(K/256), rows rounded up to even, 8] required")
    return scales.reshape(scales.shape[0], -1, 2, 4).permute(1, 0, 3, 2).reshape(scales.shape[1], -1)[:rows, :K // 32].contiguous()


def mxfp4_matmul(codes, scales, weight, weight_scales, *, bias=None, out_dtype=torch.bfloat16, activation=None,
                 residual=None, gate_table=None, indices=None):
    """[..., N]: rows of packed activations [..., K/2] times packed weights [N, K/2], each with its scales
    (quantize_mxfp4's or pack_scales', zeros in the padding), summed in fp32,
    plus bias [N] (BF16/F16/F32); its GELU-tanh with activation "gelu_tanh".  With residual BF16 of the output's
    shape, gate_table BF16 [T, N] and indices int64 [S]: residual + gate_table[indices[position]] * that
    (S: the rows' last leading dimension, or a divisor of the rows).  Every form is rounded once, from fp32."""
    _inference_only(bias, residual, gate_table)
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unsupported activation {activation!r}")
    shape = (*codes.shape[:-1], weight.shape[0])
    if codes.dim() != 2:
        codes = codes.reshape(-1, codes.shape[-1]) if codes.numel() else codes.new_empty((0, codes.shape[-1]))
    if residual is not None:
        if tuple(residual.shape) != shape:
            raise ValueError("mxfp4_matmul: a residual of the output's shape required")
        if len(shape) > 2 and indices is not None and tuple(indices.shape) != (shape[-2],):
            raise ValueError("mxfp4_matmul: int64 indices [S] required")
        residual = residual.reshape(-1, shape[-1])
    out = _matmul(codes, scales, weight, weight_scales, bias, out_dtype, _ACTIVATIONS[activation], residual, gate_table, indices)
    return out if len(shape) == 2 else out.reshape(shape)


class MXFP4Linear(nn.Module):
    """A projection in 4 bits: weights packed once (on the device they came from), activations quantized per call.
    weight BF16/F16 [N, K], N a multiple of 16, K of 32.  `weight_rounding` and `rounding` choose the scales of
    weights and activations, `activation` "gelu_tanh" the epilogue.  With `cast_float32` a float32 input is taken as BF16,
    as WeightQuantLinearModule takes it (refused without)."""

    cast_float32 = False

    def __init__(self, weight, bias=None, *, activation=None, weight_rounding="ceil", rounding="ceil", cast_float32=False):
        super().__init__()
        if not self.fits(weight.shape):
            raise ValueError("MXFP4Linear requires [N, K] with N a multiple of 16 and K of 32")
        packed, scales = quantize_mxfp4(_device_weight(weight), rounding=weight_rounding)
        self._keep(packed.to(weight.device), scales.to(weight.device), bias, activation, rounding, cast_float32)

    def _keep(self, packed, scales, bias, activation, rounding, cast_float32):
        if activation not in _ACTIVATIONS:
            raise ValueError(f"unsupported activation {activation!r}")
        _rounding(rounding)
        self.out_features, self.in_features = packed.shape[0], packed.shape[1] * 2
        if bias is not None and tuple(bias.shape) != (self.out_features,):
            raise ValueError("MXFP4Linear: bias [N] required")
        self.register_buffer("weight", packed)
        self.register_buffer("weight_scales", scales)
        self.register_buffer("bias", bias.detach().clone() if bias is not None else None)
        self.activation, self.rounding, self.cast_float32 = activation, rounding, bool(cast_float32)

    @staticmethod
    def fits(shape):
        """Whether a weight of this shape has a 4-bit form."""
        return len(shape) == 2 and shape[0] > 0 and shape[1] > 0 and shape[0] % 16 == 0 and shape[1] % 32 == 0

    @classmethod
    def from_packed(cls, weight, scales, bias=None, *, activation=None, rounding="ceil", cast_float32=False):
        """Weights packed elsewhere: codes uint8 [N, K/2] and scale bytes [N, K/32], kept as they are."""
        if weight.dtype != torch.uint8 or weight.ndim != 2 or weight.shape[0] % 16 or weight.shape[1] % 16:
            raise ValueError("MXFP4Linear.from_packed requires uint8 codes [N, K/2] with N a multiple of 16 and K of 32")
        if tuple(scales.shape) != (weight.shape[0], weight.shape[1] // 16):
            raise ValueError("MXFP4Linear.from_packed requires one scale byte per 32 values, [N, K/32]")
        result = cls.__new__(cls)
        nn.Module.__init__(result)
        result._keep(weight.contiguous(), pack_scales(scales), bias, activation, rounding, cast_float32)
        return result

    def _cast(self, x):
        return x.to(torch.bfloat16) if self.cast_float32 and x.dtype == torch.float32 else x

    def quantize_input(self, x):
        return quantize_mxfp4(self._cast(x), rounding=self.rounding)

    def forward(self, x):
        x = self._cast(x)
        if x.dtype not in (torch.bfloat16, torch.float16) or x.shape[-1] != self.in_features:
            raise ValueError(f"MXFP4Linear requires a BF16/FP16 [..., {self.in_features}] input")
        return self.forward_quantized(*self.quantize_input(x), out_dtype=x.dtype)

    def forward_quantized(self, codes, scales, out_dtype=torch.bfloat16):
        """The product of rows that are quantized already (several projections of one input): forward's result for
        quantize_input's rows; quantize_mxfp4's default rounds the scales otherwise than a module's."""
        return mxfp4_matmul(codes, scales, self.weight, self.weight_scales, bias=self.bias, out_dtype=out_dtype,
                            activation=self.activation)

    def forward_gate_residual(self, x, residual, gate_table, indices):
        """`residual + gate_table[indices] * self(x)`, rounded once, in the product's epilogue.
        x BF16/F16 [B, S, K]; residual BF16 [B, S, N]; gate_table BF16 [T, N]; indices int64 [S]."""
        if self.activation not in (None, "none"):
            raise ValueError("forward_gate_residual needs no activation")
        if x.dim() != 3 or tuple(residual.shape) != (*x.shape[:-1], self.out_features):
            raise ValueError("forward_gate_residual: x [B,S,K] and residual [B,S,N] required")
        return mxfp4_matmul(*self.quantize_input(x), self.weight, self.weight_scales, bias=self.bias, residual=residual,
                            gate_table=gate_table, indices=indices)

    def extra_repr(self):
        return (f"in_features={self.in_features}, out_features={self.out_features}, activation={self.activation}, "
                f"rounding={self.rounding}")
