"""CPU: the frequencies of rotary positions, and what the call refuses."""
import ctypes
import math

import numpy as np
import pytest

from pkgpu import pk
from test_decode_refusals import refused


def freqs(rot, base, scaling=0, factor=1.0, trained=0.0, slow=0.0, fast=0.0):
    out = np.full(rot // 2 + 1, 7.0, np.float32)
    pk.call("pk_gpu_rope_freqs", rot, base, scaling, factor, trained, slow, fast, out.ctypes.data)
    assert out[-1] == 7.0
    return out[:-1].astype(np.float64)


@pytest.mark.parametrize("rot", [2, 4, 6, 64, 128, 1024])
@pytest.mark.parametrize("base", [10000.0, 500000.0, 0.5])
def test_against_the_formulas(rot, base):
    i = np.arange(rot // 2)
    f = base ** (-2.0 * i / rot)
    near = dict(rtol=2.0 ** -24 * 1.001, atol=0)
    np.testing.assert_allclose(freqs(rot, base), f, **near)
    np.testing.assert_allclose(freqs(rot, base, pk.ROPE_LINEAR, 4.0), f / 4, **near)
    if rot > 2:
        got = freqs(rot, base, pk.ROPE_BASE, 8.0)
        np.testing.assert_allclose(got, (base * 8.0 ** (rot / (rot - 2))) ** (-2.0 * i / rot), **near)
        assert got[0] == 1.0 and math.isclose(got[-1], f[-1] / 8, rel_tol=1e-6)
    turns = 4096 * f / (2 * math.pi)
    keep = np.clip((turns - 1) / 31, 0, 1)
    np.testing.assert_allclose(freqs(rot, base, pk.ROPE_PARTS, 8.0, 4096.0, 1.0, 32.0), f * keep + f / 8 * (1 - keep), **near)


GOOD = dict(rot=64, base=1e4, scaling=pk.ROPE_PARTS, factor=8.0, trained=4096.0, slow=1.0, fast=32.0)


@pytest.mark.parametrize("kw,text", [
    (dict(rot=0), "rot_dim"), (dict(rot=63), "rot_dim"), (dict(rot=-2), "rot_dim"), (dict(rot=1026), "rot_dim"),
    (dict(base=0.0), "base"), (dict(base=math.nan), "base"), (dict(base=math.inf), "base"), (dict(scaling=4), "scaling"),
    (dict(scaling=-1), "scaling"), (dict(factor=0.0), "factor"), (dict(factor=math.nan), "factor"),
    (dict(factor=math.inf, scaling=pk.ROPE_LINEAR), "factor"), (dict(rot=2, scaling=pk.ROPE_BASE), "rot_dim"),
    (dict(trained=0.0), "trained"), (dict(slow=-1.0), "slow"), (dict(fast=1.0), "fast"), (dict(fast=math.inf), "fast"),
])
def test_refusals(kw, text):
    d = dict(GOOD, **kw)
    out = np.zeros(2048, np.float32)
    refused("pk_gpu_rope_freqs", *d.values(), out.ctypes.data, text=text)
    assert not out.any()


def test_no_memory_for_them():
    refused("pk_gpu_rope_freqs", *GOOD.values(), None, text="NULL")
    assert ctypes.sizeof(pk.Rope) == 24
