"""rotary_frequencies against restatements of the published scalings, pair by pair, and its refusals."""
import math

import pytest

from xgen_amd.operator.qk_norm_rope import rotary_frequencies


@pytest.mark.parametrize("dim,base,factor,length,low,high", [(128, 500000.0, 8.0, 8192, 1.0, 4.0), (64, 500000.0, 32.0, 8192, 1.0, 4.0), (96, 1e4, 2.0, 4096, 1.5, 16.0)])
def test_bands(dim, base, factor, length, low, high):
    """Rope type "llama3": by wavelengths, as it is published."""
    got, scale = rotary_frequencies(dim, base=base, scaling="bands", factor=factor, trained_length=length, low=low, high=high)
    for i in range(dim // 2):
        f = base ** (-2 * i / dim)
        wave = 2 * math.pi / f
        if wave > length / low:
            want = f / factor
        elif wave < length / high:
            want = f
        else:
            smooth = (length / wave - low) / (high - low)
            want = (1 - smooth) * f / factor + smooth * f
        assert abs(float(got[i]) / want - 1) < 1e-13, i
    assert scale == 1.0


@pytest.mark.parametrize("dim,base,factor,length,slow,fast", [(128, 1e4, 4.0, 4096, 1.0, 32.0), (64, 1e6, 40.0, 4096, 1.0, 32.0), (128, 1e4, 16.0, 512, 1.0, 32.0)])
def test_ramp(dim, base, factor, length, slow, fast):
    """YaRN: interpolated and plain frequencies blended by a ramp between two whole pairs."""
    got, scale = rotary_frequencies(dim, base=base, scaling="ramp", factor=factor, trained_length=length, low=slow, high=fast)

    def pair(turns):
        return dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(base))
    first, last = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), dim - 1)
    for i in range(dim // 2):
        ramp = min(max((i - first) / max(last - first, 0.001), 0), 1)
        f = base ** (-2 * i / dim)
        want = f / factor * ramp + f * (1 - ramp)
        assert abs(float(got[i]) / want - 1) < 1e-13, i
    assert scale == 0.1 * math.log(factor) + 1


@pytest.mark.parametrize("scaling", ["bands", "ramp"])
@pytest.mark.parametrize("length", [0, -4096, float("nan")])
def test_refused_lengths(scaling, length):
    with pytest.raises(ValueError, match="trained_length"):
        rotary_frequencies(64, scaling=scaling, factor=2.0, trained_length=length)
