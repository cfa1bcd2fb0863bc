"""MXFP4Linear and its installer without a GPU: which inputs an installed module takes, and what the installer refuses."""
import pytest
import torch

from xgen_amd.operator import mxfp4

BF, HF, F32, U8, I64 = torch.bfloat16, torch.float16, torch.float32, torch.uint8, torch.int64


def module(n=16, k=64, **kw):
    w, s = torch.zeros((n, k // 2), dtype=U8, device="meta"), torch.zeros((n, k // 32), dtype=U8, device="meta")
    return mxfp4.MXFP4Linear.from_packed(w, s, **kw)


def test_float32_inputs_are_cast_where_asked_for():
    x, linear = torch.zeros((2, 3, 64), device="meta"), module(cast_float32=True)
    out = linear(x)
    assert out.dtype == BF and out.shape == (2, 3, 16)
    assert linear(x.to(HF)).dtype == HF and linear(x.to(BF)).dtype == BF
    assert linear.quantize_input(x)[0].shape == (2, 3, 32)
    t = torch.zeros((2, 3, 16), dtype=BF, device="meta")
    gated = linear.forward_gate_residual(x, t, t[0], torch.zeros(3, dtype=I64, device="meta"))
    assert gated.dtype == BF and gated.shape == t.shape
    with pytest.raises(ValueError, match="input"):
        linear(x.double())
    with pytest.raises(ValueError, match="input"):
        module()(x)
