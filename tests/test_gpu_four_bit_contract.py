"""The operators of the 4-bit path: their Meta functions and native checks accept and refuse the same calls
(tests/test_gpu_contract.py's form)."""
import pytest
import torch

import xgen_amd  # noqa: F401
from test_experts_cpu import outcome
from test_four_bit_cpu import ACCEPTED, REFUSED

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", sorted(ACCEPTED))
def test_accepted_alike(cuda, name):
    meta, device = outcome(ACCEPTED[name], "meta"), outcome(ACCEPTED[name], cuda)
    torch.cuda.synchronize()
    assert meta[0] == "accepted" and device == meta


@pytest.mark.parametrize("name", sorted(REFUSED))
def test_refused_alike(cuda, name):
    meta, device = outcome(REFUSED[name], "meta"), outcome(REFUSED[name], cuda)
    assert meta[0] == "refused" and device == meta
