"""CPU: what the rotary calls refuse, before any device is touched.  Pointers here are
small aligned numbers that nothing may dereference."""
import ctypes

import pytest

from pkgpu import gpu_available, pk
from test_decode_refusals import BAD_CACHES, P, cache, refused


def rope(**kw):
    d = dict(freqs=P, scale=1.0, rot_dim=64, interleaved=0)
    d.update(kw)
    return ctypes.byref(pk.Rope(*d.values()))


def rows(code=-1, text=None, **kw):
    d = dict(r=rope(), dtype=pk.BF16, x=P, ldx=512, heads=4, dim=128, pos=P, n=3, y=P, ldy=512)
    d.update(kw)
    refused("pk_gpu_rope_dev", *d.values(), None, code=code, text=text)


def write(code=-1, text=None, **kw):
    d = dict(r=rope(), c=ctypes.byref(cache()), dtype=pk.BF16, q=P, ldq=512, heads=4, qo=P, ldqo=512, k=P, ldk=256, v=P,
             ldv=256, pos=P, slots=P, n=3)
    d.update(kw)
    refused("pk_gpu_rope_kv_write_dev", *d.values(), None, code=code, text=text)


BAD_ROPES = [(dict(rot_dim=0), "rot_dim"), (dict(rot_dim=63), "rot_dim"), (dict(rot_dim=130), "rot_dim"),
             (dict(rot_dim=-2), "rot_dim"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
             (dict(freqs=None), "NULL freq"), (dict(freqs=P + 2), "aligned")]


@pytest.mark.parametrize("kw,text", BAD_ROPES)
def test_bad_ropes(kw, text):
    rows(r=rope(**kw), text=text)
    write(r=rope(**kw), text=text)


def test_null_ropes():
    rows(r=None, text="NULL rope")
    write(r=None, text="NULL rope")
    write(c=None, text="NULL cache")


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=pk.I8), -1, "type"), (dict(dtype=pk.E2M1), -1, "type"), (dict(ldx=511), -1, "ldx"), (dict(ldy=511), -1, "ldy"),
    (dict(heads=-1), -1, "heads"), (dict(dim=1), -2, "head_dim"), (dict(dim=1026), -2, "head_dim"), (dict(n=-1), -1, "n ="),
    (dict(x=None), -1, "NULL"), (dict(y=None), -1, "NULL"), (dict(pos=None), -1, "NULL"), (dict(x=P + 1), -1, "aligned"),
    (dict(y=P + 1), -1, "aligned"), (dict(pos=P + 2), -1, "aligned"), (dict(ldx=520), -1, "in place"),
    (dict(heads=1 << 25), -1, "elements"),
])
def test_bad_rows(kw, code, text):
    rows(code=code, text=text, **kw)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=pk.E4M3), "type"), (dict(ldq=511), "ldq"), (dict(ldqo=511), "ldqo"), (dict(ldk=255), "ldk"),
    (dict(ldv=255), "ldv"), (dict(heads=-1), "heads"), (dict(n=-1), "n ="), (dict(q=None), "NULL"), (dict(qo=None), "NULL"),
    (dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(pos=None), "NULL"), (dict(slots=None), "NULL"),
    (dict(q=P + 8), "aligned"), (dict(qo=P + 8), "aligned"), (dict(k=P + 8), "aligned"), (dict(v=P + 4), "aligned"),
    (dict(ldk=260), "aligned"), (dict(ldqo=516), "aligned"), (dict(pos=P + 2), "aligned"), (dict(slots=P + 1), "aligned"),
    (dict(ldq=520), "in place"), (dict(n=1 << 30), "2^31"), (dict(heads=1 << 25, ldq=1 << 30, ldqo=1 << 30), "elements"),
])
def test_bad_writes(kw, text):
    write(text=text, **kw)


@pytest.mark.parametrize("bad,code,text", BAD_CACHES)
def test_bad_caches(bad, code, text):
    write(c=ctypes.byref(cache(**bad)), ldk=1 << 30, ldv=1 << 30, code=code, text=text)


def test_4_bit_caches_need_their_bytes():
    for name in ("k_scale", "v_scale"):
        write(c=ctypes.byref(cache(dtype=pk.E2M1, **{name: None})), text="NULL")


@pytest.mark.skipif(gpu_available(), reason="checks the no-device error path")
def test_no_device_is_an_error():
    for n in (0, 3):
        rows(n=n, code=-5)
        write(n=n, code=-5)
        write(n=n, heads=0, q=None, qo=None, ldq=0, ldqo=0, code=-5)
    rows(n=(1 << 24) - 1, heads=1, ldx=128, ldy=128, code=-5)
