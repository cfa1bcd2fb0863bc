"""What the C entries of a block with experts refuse at the edges of their ranges, before any HIP call."""
import pytest

from test_experts_cpu import GROUPED, NO, call
from xgen_amd import _native as N


def refused(fn, good, changes, status, needle):
    L = N.lib()
    assert call(fn, good, **changes)(L) == status, L.xgen_last_error()
    assert needle in L.xgen_last_error()


@pytest.mark.parametrize("bias", [18, 20, 24])
@pytest.mark.parametrize("dtype", [N.DTYPE_BF16, N.DTYPE_F16, N.DTYPE_F32])
def test_unaligned_bias(built_library, bias, dtype):
    refused("xgen_grouped_matmul", GROUPED, dict(bias=bias, bdt=dtype), NO, b"bias must be 16-byte aligned")
