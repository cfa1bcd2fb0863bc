"""MXFP4Linear as a model's layers use it (tests/test_gpu_mxfp4.py has its product)."""
import pytest
import torch

import xgen_amd  # noqa: F401
from test_gpu_mxfp4 import check_product, gated_inputs, rows
from xgen_amd.config import QuantLayerConfig
from xgen_amd.operator.matmul import enable_weight_quant_linear
from xgen_amd.operator.mxfp4 import MXFP4Linear, quantize_mxfp4

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def test_installed_in_a_float32_model(cuda):
    """Float32 weights, biases and activations: what the 8-bit installer's modules take."""
    torch.manual_seed(1)
    layers = [torch.nn.Linear(64, 96), torch.nn.GELU(), torch.nn.Linear(96, 32)]
    w = quantize_mxfp4(layers[0].weight.data.to(BF).to(cuda), rounding="ceil")
    bias = layers[0].bias.data.to(cuda)
    model = enable_weight_quant_linear(torch.nn.Sequential(*layers), QuantLayerConfig(), dtype="mxfp4").to(cuda)
    assert isinstance(model[0], MXFP4Linear) and isinstance(model[2], MXFP4Linear)
    x = rows(torch.Generator().manual_seed(2), 5, 64, F32).to(cuda)
    assert x.dtype == F32 and model(x).shape == (5, 32)
    got = model[0](x)
    check_product(quantize_mxfp4(x.to(BF), rounding="ceil"), w, 5, 96, 64, bias, got=got)
    assert torch.equal(got, model[0](x.to(BF)))
    res, gate, idx = gated_inputs(torch.Generator().manual_seed(3), cuda, 5, 96, 4, 5)
    res = res[None]
    assert torch.equal(model[0].forward_gate_residual(x[None], res, gate, idx), model[0].forward_gate_residual(x[None].to(BF), res, gate, idx))


@pytest.mark.parametrize("rounding", [None, "floor", "ceil"])
def test_shared_rows(cuda, rounding):
    """Rows that a module quantized give its own result through it and through every other of its rounding."""
    g = torch.Generator().manual_seed(4)
    kw = {} if rounding is None else {"rounding": rounding}
    up, gate = (MXFP4Linear((torch.randn((96, 160), generator=g) * 0.02).to(BF).to(cuda), activation=a, **kw) for a in ("gelu_tanh", None))
    x = torch.randn((2, 70, 160), generator=g).to(BF).to(cuda)
    shared = up.quantize_input(x)
    for linear in (up, gate):
        assert torch.equal(linear.forward_quantized(*shared), linear(x))
    other = quantize_mxfp4(x, rounding="floor" if rounding != "floor" else "ceil")
    assert not torch.equal(up.forward_quantized(*other), up(x))
