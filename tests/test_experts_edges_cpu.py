"""What the operators of a block with experts and their C entries refuse at the edges of their ranges, before any HIP
call (tests/test_gpu_experts_edges.py makes the operators' calls on the device)."""
import pytest

from test_experts_cpu import BAD, COMBINE, GROUPED, NO, NORM, call, norm, outcome
from xgen_amd import _native as N


def refused(fn, good, changes, status, needle):
    L = N.lib()
    assert call(fn, good, **changes)(L) == status, L.xgen_last_error()
    assert needle in L.xgen_last_error()


@pytest.mark.parametrize("bias", [18, 20, 24])
@pytest.mark.parametrize("dtype", [N.DTYPE_BF16, N.DTYPE_F16, N.DTYPE_F32])
def test_unaligned_bias(built_library, bias, dtype):
    refused("xgen_grouped_matmul", GROUPED, dict(bias=bias, bdt=dtype), NO, b"bias must be 16-byte aligned")


# (1.1754943e-38 is 2^-126 as a float32: a third of its step of 2^-149 away)
EPS_TAKEN = [2.0 ** -126, 1.1754943e-38, 1.2e-38, 1e-30, 0.5, 1 - 2.0 ** -24]
# below what the kernel's reciprocal square root takes for a number; 0 and 1 as a float32
EPS_REFUSED = [2.0 ** -126 - 2.0 ** -149, 1e-38, 1e-40, 1e-45, 1e-46, -1e-6, 1 - 1e-9, float("nan"), float("inf")]


@pytest.mark.parametrize("eps", EPS_TAKEN)
def test_eps_taken(eps):
    assert outcome(norm(eps=eps), "meta")[0] == "accepted"


@pytest.mark.parametrize("eps", EPS_REFUSED)
def test_eps_refused(built_library, eps):
    assert outcome(norm(eps=eps), "meta") == ("refused", "residual_norm: eps must be in [2^-126, 1) as a float32")
    refused("xgen_residual_norm", NORM, dict(eps=eps), BAD, b"eps")


@pytest.mark.parametrize("M", [2 ** 31 - 256, 2 ** 31 - 1, 2 ** 31])
def test_more_grouped_rows_than_are_counted(built_library, M):
    refused("xgen_grouped_matmul", GROUPED, dict(M=M, ar=M, N=16, G=1, ldo=16), NO, b"too many rows")
    refused("xgen_grouped_matmul", GROUPED, dict(M=M, rows=16, N=16, G=1, ldo=16), NO, b"too many rows")


@pytest.mark.parametrize("k", [2 ** 30, 2 ** 31 - 4, 2 ** 31 - 1, 2 ** 31])
def test_more_choices_than_are_counted(built_library, k):
    refused("xgen_expert_combine", COMBINE, dict(tokens=1, seq=1, k=k), NO, b"too many rows or choices")
