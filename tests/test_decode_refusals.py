"""CPU: what the decoder operators refuse, before any device is touched.

Pointers here are small aligned numbers that nothing may dereference."""
import ctypes

import pytest

from pkgpu import pk

P = 1 << 20             # an aligned address no call may read


def cache(**kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, dtype=pk.I8, n_pages=4, page_size=16, heads=2, head_dim=128)
    d.update(kw)
    return pk.KvCache(*[d[n] for n, _ in pk.KvCache._fields_])


def refused(fn, *args, code=-1, text=None):
    lib = pk.load()
    assert getattr(lib, fn)(*args) == code
    msg = lib.pk_gpu_last_error().decode()
    assert msg and (text is None or text in msg), msg


BAD_CACHES = [
    (dict(k=None), -1, "NULL"), (dict(v=None), -1, "NULL"), (dict(k_scale=None), -1, "NULL"),
    (dict(v_scale=None), -1, "NULL"), (dict(k=P + 8), -1, "aligned"), (dict(v_scale=P + 4), -1, "aligned"),
    (dict(dtype=pk.F32), -1, "type"), (dict(dtype=9), -1, "type"), (dict(head_dim=96), -2, "head_dim"),
    (dict(head_dim=0), -2, "head_dim"), (dict(page_size=8), -2, "page_size"), (dict(page_size=48), -2, "page_size"),
    (dict(page_size=0), -2, "page_size"), (dict(page_size=-16), -2, "page_size"), (dict(n_pages=0), -1, "pages"),
    (dict(heads=0), -1, "heads"), (dict(n_pages=1 << 28), -1, "2^31"), (dict(heads=1 << 25), -1, "2^31"),
]


@pytest.mark.parametrize("bad,code,text", BAD_CACHES)
def test_bad_caches(bad, code, text):
    c = ctypes.byref(cache(**bad))
    refused("pk_gpu_kv_write_dev", c, pk.F32, P, 1 << 30, P, 1 << 30, P, 1, None, code=code, text=text)
    refused("pk_gpu_kv_read_dev", c, pk.F32, P, 1, P, 1 << 30, P, 1 << 30, None, code=code, text=text)


def test_16_bit_caches_need_no_scales():
    c = cache(dtype=pk.BF16, k_scale=None, v_scale=None)
    refused("pk_gpu_kv_write_dev", ctypes.byref(c), pk.F32, None, 256, P, 256, P, 1, None, text="NULL operand")


@pytest.mark.parametrize("dtype,k,ldk,v,ldv,slots,n,text", [
    (pk.I8, P, 256, P, 256, P, 1, "type"), (-1, P, 256, P, 256, P, 1, "type"),
    (pk.F32, P, 255, P, 256, P, 1, "ldk"), (pk.F32, P, 256, P, 0, P, 1, "ldv"),
    (pk.F32, P, 256, P, 256, P, -1, "n ="), (pk.F32, None, 256, P, 256, P, 1, "NULL"),
    (pk.F32, P, 256, None, 256, P, 1, "NULL"), (pk.F32, P, 256, P, 256, None, 1, "NULL"),
    (pk.F32, P + 4, 256, P, 256, P, 1, "aligned"), (pk.BF16, P, 256, P, 260, P, 1, "aligned"),
    (pk.F32, P, 256, P, 256, P, 1 << 30, "2^31"),
])
def test_bad_rows(dtype, k, ldk, v, ldv, slots, n, text):
    c = ctypes.byref(cache())
    refused("pk_gpu_kv_write_dev", c, dtype, k, ldk, v, ldv, slots, n, None, text=text)
    refused("pk_gpu_kv_read_dev", c, dtype, slots, n, k, ldk, v, ldv, None, text=text)


def test_null_cache():
    refused("pk_gpu_kv_write_dev", None, pk.F32, P, 256, P, 256, P, 1, None, text="NULL cache")
    refused("pk_gpu_kv_read_dev", None, pk.F32, P, 1, P, 256, P, 256, None, text="NULL cache")
