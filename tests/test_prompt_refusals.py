"""CPU: what the attention with rules refuses, its workspaces and its launches' limits, before
any device is touched.  Pointers here are small aligned numbers that nothing may dereference."""
import ctypes
import re

import pytest

from pkgpu import gpu_available, pk
from test_decode_refusals import BAD_CACHES, P, cache, refused


def rules(**kw):
    d = dict(scale=1.0, cap=0.0, slopes=None, window=0, first=None, until=None)
    d.update(kw)
    return ctypes.byref(pk.AttentionRules(*d.values()))


def attention(code=-1, text=None, **kw):
    d = dict(c=ctypes.byref(cache()), dtype=pk.BF16, q=P, ldq=512, heads=4, pages=P, ld_pages=8, lens=P, starts=P, B=3,
             rows=30, max_new=10, max_len=128, rules=rules(), out=P, ldo=512, lse=None, ws=P, floats=1 << 40)
    d.update(kw)
    refused("pk_gpu_prompt_attention_dev", *d.values(), None, code=code, text=text)


@pytest.mark.parametrize("kw,code,text", [
    (dict(rules=None), -1, "NULL rules"), (dict(c=None), -1, "NULL cache"), (dict(dtype=pk.I8), -1, "type"),
    (dict(dtype=pk.E2M1), -1, "type"), (dict(heads=0), -1, "heads"), (dict(heads=3), -1, "heads"), (dict(B=-1), -1, "B ="),
    (dict(rows=-1), -1, "rows"), (dict(max_new=-1), -1, "max_new"), (dict(max_len=-1), -1, "max_len"),
    (dict(max_len=(1 << 30) + 1), -1, "2^30"), (dict(max_new=(1 << 30) + 1), -1, "2^30"),
    (dict(rules=rules(window=-1)), -1, "window"), (dict(rules=rules(scale=float("nan"))), -1, "scale"),
    (dict(rules=rules(scale=float("inf"))), -1, "scale"), (dict(rules=rules(cap=-1.0)), -1, "cap"),
    (dict(rules=rules(cap=float("nan"))), -1, "cap"), (dict(rules=rules(cap=float("inf"))), -1, "cap"),
    (dict(rules=rules(scale=1.5e36)), -1, "scale"), (dict(rules=rules(cap=1.5e36)), -1, "cap"),
    (dict(rules=rules(scale=-1.5e36)), -1, "scale"), (dict(rules=rules(scale=1.0, cap=1e-37)), -1, "cap"),
    (dict(ldq=511), -1, "ldq"), (dict(ldo=511), -1, "ldo"), (dict(ld_pages=7), -1, "pages"), (dict(ld_pages=-1), -1, "pages"),
    (dict(q=None), -1, "NULL"), (dict(out=None), -1, "NULL"), (dict(lens=None), -1, "NULL"), (dict(pages=None), -1, "NULL"),
    (dict(q=P + 8), -1, "aligned"), (dict(out=P + 4), -1, "aligned"), (dict(ldq=514), -1, "aligned"),
    (dict(ldo=516), -1, "aligned"), (dict(pages=P + 1), -1, "aligned"), (dict(lens=P + 2), -1, "aligned"),
    (dict(starts=P + 2), -1, "aligned"), (dict(lse=P + 3), -1, "aligned"), (dict(rules=rules(slopes=P + 1)), -1, "aligned"),
    (dict(rules=rules(first=P + 2)), -1, "aligned"), (dict(rules=rules(until=P + 2)), -1, "aligned"),
    (dict(B=1 << 30, rows=1 << 30), -1, "grid"),
])
def test_bad_calls(kw, code, text):
    attention(code=code, text=text, **kw)


@pytest.mark.parametrize("bad,code,text", BAD_CACHES)
def test_bad_caches(bad, code, text):
    c = ctypes.byref(cache(**bad))
    heads = 1 << 25 if bad.get("heads") else 2
    attention(c=c, ldq=1 << 30, ldo=1 << 30, heads=heads, code=code, text=text)
    assert pk.load().pk_gpu_prompt_attention_ws_floats(c, 1, 1, heads, 1, 1000, 0) == 0


@pytest.mark.parametrize("held,dtype", [(pk.F16, pk.F32), (pk.F16, pk.BF16), (pk.BF16, pk.F16)])
def test_queries_a_16_bit_cache_does_not_take(held, dtype):
    attention(c=ctypes.byref(cache(dtype=held)), dtype=dtype, code=-2, text="queries")


def query(c, B, rows, heads, max_new, max_len, window):
    return pk.load().pk_gpu_prompt_attention_ws_floats(ctypes.byref(c), B, rows, heads, max_new, max_len, window)


def needed(c, B, rows, heads, max_new, max_len, window, dtype=pk.BF16, starts=P):
    """Floats that a call asks for: what its refusal of no workspace names; 0 where it gets as far as the device, or is too large."""
    lib = pk.load()
    wide = heads * c.head_dim
    rc = lib.pk_gpu_prompt_attention_dev(ctypes.byref(c), dtype, P, wide, heads, P, 1 << 30, P, starts, B, rows, max_new, max_len,
                                         rules(window=window), P, wide, None, None, 0, None)
    if rc == -5:
        return 0
    assert rc == -1
    text = lib.pk_gpu_last_error().decode()
    return 0 if "grid" in text else int(re.search(r"workspace of (\d+) floats", text).group(1))


no_gpu = pytest.mark.skipif(gpu_available(), reason="makes calls with addresses that nothing may read")


@no_gpu
@pytest.mark.parametrize("kind,heads,group,dim", [(pk.I8, 8, 4, 128), (pk.BF16, 2, 1, 256), (pk.E4M3, 1, 20, 64),
                                                  (pk.E2M1, 3, 5, 128), (pk.F16, 1, 1, 64), (pk.BF16, 32, 1, 128)])
def test_a_workspace_is_enough_for_every_smaller_call(kind, heads, group, dim):
    """Walked over B, max_new, max_len and window: the query never falls, and covers what calls ask for."""
    c = cache(dtype=kind, heads=heads, head_dim=dim, n_pages=1 << 20)
    before = {}
    lengths = (1, 700, 769, 2304, 8192, 8193, 30000, 100000, 1 << 20, 1 << 30)
    for n, length in enumerate(lengths):
        for i, B in enumerate((1, 2, 3, 5, 8, 31, 64, 256, 600)):
            for j, new in enumerate((1, 2, 5, 16, 17, 33, 64, 65, 128, 129, 300, 1000, 5000, 70000)):
                for k, w in enumerate((1, 700, 5000, 0)):
                    rows = min(B * new, 1 << 30)
                    got = query(c, B, rows, heads * group, new, length, w)
                    asked = [needed(c, B, rows, heads * group, new, length, w, dtype=t)
                             for t in ((pk.F16,) if kind == pk.F16 else (pk.BF16, pk.F32))]
                    assert got >= max(asked)
                    for at in ((n - 1, i, j, k), (n, i - 1, j, k), (n, i, j - 1, k), (n, i, j, k - 1)):
                        assert got >= before.get(at, 0)
                    before[n, i, j, k] = got


@no_gpu
def test_a_workspace_that_is_too_small():
    c = cache(n_pages=1 << 20)
    for new in (1, 5, 100, 1000):
        need = needed(c, 1, new, 4, new, 100000, 0)
        assert 0 < need <= query(c, 1, new, 4, new, 100000, 0)
        for ws, floats in ((None, need), (P, need - 1), (P + 4, need)):
            attention(c=ctypes.byref(c), B=1, rows=new, max_new=new, max_len=100000, ld_pages=6250, ws=ws, floats=floats,
                      text="workspace")
    assert needed(c, 3, 30, 4, 10, 128, 0) == 0


@no_gpu
def test_no_device_is_an_error():
    for kw in (dict(), dict(B=0), dict(rows=0), dict(max_new=0), dict(starts=None), dict(max_len=0, pages=None, ld_pages=0)):
        attention(code=-5, **kw)
