"""MXFP4Linear and its installer without a GPU: which inputs an installed module takes, and what the installer refuses."""
import pytest
import torch
from torch import nn

from test_experts_cpu import call
from test_four_bit_cpu import MM
from xgen_amd import _native as N
from xgen_amd.config import QuantLayerConfig
from xgen_amd.operator import matmul, mxfp4

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


@pytest.mark.parametrize("last", [nn.Linear(96, 24), nn.Linear(48, 32), nn.Linear(96, 32, dtype=torch.float64)])
def test_installer_refuses_before_it_replaces(last):
    """A layer without a 4-bit form: named, and the layers before it are as they were."""
    model = nn.Sequential(nn.Linear(64, 96), nn.Sequential(nn.GELU(), last))
    with pytest.raises(ValueError, match=r"exclude.*: 1\.1 \("):
        matmul.enable_weight_quant_linear(model, QuantLayerConfig(), dtype="mxfp4")
    assert type(model[0]) is nn.Linear and model[1][1] is last
    with pytest.raises(ValueError) as error:
        matmul.matmul_manager.enable_online_dynamic_quant(model, QuantLayerConfig(), dtype="mxfp4")
    assert "1.1 (" in str(error.value.__cause__)


def test_installer_excludes_what_does_not_fit():
    model = nn.Sequential(nn.Linear(96, 24), nn.ReLU())
    config = QuantLayerConfig(exclude_patterns=["0"])
    assert matmul.enable_weight_quant_linear(model, config, dtype="mxfp4") is model and type(model[0]) is nn.Linear


@pytest.mark.parametrize("dtype", ["w8a8", "mxfp4"])
def test_the_installer_logs_what_it_installs(dtype, caplog):
    with caplog.at_level("INFO", logger=matmul.LOG.name):
        matmul.matmul_manager.enable_online_dynamic_quant(nn.Sequential(nn.ReLU()), QuantLayerConfig(), dtype=dtype)
        with pytest.raises(ValueError):
            matmul.matmul_manager.enable_online_dynamic_quant(nn.Sequential(nn.Linear(48, 24, dtype=torch.float64)), QuantLayerConfig(), dtype=dtype)
    said = [r.getMessage() for r in caplog.records]
    assert len(said) == 4 and all(dtype.upper() in m for m in said), said
    assert "installed" in said[1] and "failed" in said[3]


def test_longest_sequence_of_a_gated_product(built_library):
    L = N.lib()
    rows = 1 << 28
    assert call("xgen_mxfp4_matmul", MM, M=rows, seq=rows, ab=rows * 8)(L) == N.ERR_UNSUPPORTED
    assert b"2^28" in L.xgen_last_error()
