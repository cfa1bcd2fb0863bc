"""The new operators' Meta functions and native checks accept and refuse the same calls (tests/test_gpu_contract.py's
form): every call on meta tensors and on the device gives the same shapes, strides and dtypes, or the same error."""
import pytest
import torch

import xgen_amd  # noqa: F401
from test_experts_cpu import ACCEPTED, REFUSED, outcome

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", sorted(ACCEPTED))
def test_accepted_alike(cuda, name):
    meta, device = outcome(ACCEPTED[name], "meta"), outcome(ACCEPTED[name], cuda)
    assert meta[0] == "accepted" and device == meta


@pytest.mark.parametrize("name", sorted(REFUSED))
def test_refused_alike(cuda, name):
    meta, device = outcome(REFUSED[name], "meta"), outcome(REFUSED[name], cuda)
    assert meta[0] == "refused" and device == meta
