"""CPU: bases and factors whose frequencies a float does not hold are refused, before any is written;
frequencies too small for one are 0."""
import numpy as np
import pytest

from pkgpu import pk
from test_decode_refusals import refused
from test_rope_freqs import freqs


@pytest.mark.parametrize("args", [
    (128, 1e-300, pk.ROPE_PLAIN, 1.0, 0.0, 0.0, 0.0), (128, 1e4, pk.ROPE_LINEAR, 1e-300, 0.0, 0.0, 0.0),
    (2, 1e4, pk.ROPE_LINEAR, 1e-39, 0.0, 0.0, 0.0), (128, 1e200, pk.ROPE_BASE, 1e200, 0.0, 0.0, 0.0),
    (128, 1e-200, pk.ROPE_BASE, 1e-200, 0.0, 0.0, 0.0), (128, 1e4, pk.ROPE_PARTS, 1e-200, 4096.0, 1.0, 32.0),
])
def test_frequencies_past_a_float(args):
    out = np.full(64, 7.0, np.float32)
    refused("pk_gpu_rope_freqs", *args, out.ctypes.data, text="frequencies")
    assert np.all(out == 7.0)


def test_frequencies_below_a_float():
    got = freqs(128, 1e300)
    assert got[0] == 1.0 and got[-1] == 0.0 and np.isfinite(got).all()


@pytest.mark.parametrize("rot,base,scaling,factor", [(128, 1e-30, pk.ROPE_PLAIN, 1.0), (64, 1e30, pk.ROPE_BASE, 1e8),
                                                      (2, 1.0, pk.ROPE_LINEAR, 1e-38)])
def test_the_largest_that_are_held(rot, base, scaling, factor):
    i = np.arange(rot // 2)
    b = base * factor ** (rot / (rot - 2)) if scaling == pk.ROPE_BASE else base
    want = b ** (-2.0 * i / rot) / (factor if scaling == pk.ROPE_LINEAR else 1.0)
    np.testing.assert_allclose(freqs(rot, base, scaling, factor), want, rtol=2.0 ** -24 * 1.001, atol=2.0 ** -150)


def test_turns_without_end_keep_a_frequency():
    np.testing.assert_allclose(freqs(128, 1e4, pk.ROPE_PARTS, 2.0, 1e308, 1.0, 1.0 + 1e-12), 1e4 ** (-np.arange(64) / 64.0),
                               rtol=2.0 ** -24 * 1.001)
