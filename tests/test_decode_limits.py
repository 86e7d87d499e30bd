"""CPU: sizes the decoder operators take: workspaces that are large enough for every
smaller call, and launches that would pass the device's limits, refused before
any device is touched.

Pointers here are small aligned numbers that nothing may dereference."""
import ctypes
import re

import pytest

from pkgpu import gpu_available, pk
from test_decode_refusals import P, attention, cache, gemm, refused

# calls that are not refused end without a device, and only so
pytestmark = pytest.mark.skipif(gpu_available(), reason="makes calls with addresses that nothing may read")


def needed(c, B, heads, max_len, window):
    """Floats that a call asks for: what its refusal of no workspace names; 0 where it gets as far as the device."""
    lib = pk.load()
    wide = heads * c.head_dim
    rc = lib.pk_gpu_paged_attention_dev(ctypes.byref(c), pk.BF16, P, wide, heads, P, 1 << 30, P, B, max_len, 1.0,
                                        window, P, wide, None, None, 0, None)
    if rc == -5:
        return 0
    assert rc == -1
    return int(re.search(r"workspace of (\d+) floats", lib.pk_gpu_last_error().decode()).group(1))


def query(c, B, heads, max_len, window):
    return pk.load().pk_gpu_paged_attention_ws_floats(ctypes.byref(c), B, heads, max_len, window)


LENGTHS = sorted({n + d for n in (1, 512, 768, 1024, 2048, 2304, 8192, 8448, 30000, 65536, 100000, 131072, 1 << 20, 1 << 30)
                  for d in (-1, 0, 1) if 0 < n + d <= 1 << 30})


@pytest.mark.parametrize("kind,heads,group,dim", [(pk.I8, 8, 4, 128), (pk.BF16, 2, 1, 256), (pk.E4M3, 1, 20, 64),
                                                  (pk.BF16, 3, 5, 128), (pk.I8, 1, 1, 64)])
def test_a_workspace_is_enough_for_every_smaller_call(kind, heads, group, dim):
    """Walked over max_len, B and window: the query never falls, and covers what calls ask for."""
    c = cache(dtype=kind, heads=heads, head_dim=dim, n_pages=1 << 20)
    batches = (1, 2, 3, 4, 5, 7, 8, 16, 31, 32, 33, 63, 64, 100, 255, 256, 257, 600)
    windows = (1, 700, 1000, 5000, 50000, 0)             # 0 sees all
    before = {}
    for n in LENGTHS:
        for i, B in enumerate(batches):
            for j, w in enumerate(windows):
                got = query(c, B, heads * group, n, w)
                assert got >= needed(c, B, heads * group, n, w)
                assert got >= max(before.get((i, j), 0), before.get((i - 1, j), 0), before.get((i, j - 1), 0))
                before[i, j] = got


def test_a_closer_length_takes_the_bounds_workspace():
    c = cache(n_pages=1 << 20, heads=8)
    bound = query(c, 1, 32, 1 << 20, 0)
    for n in (8192, 8193, 8448, 12000, 65536):
        assert 0 < needed(c, 1, 32, n, 0) <= bound


# Launches take below 2^32 threads: the sizes on both sides of that.

@pytest.mark.parametrize("heads,dim,n,code", [
    (1, 256, 1 << 27, -1), (1, 256, (1 << 27) - 32, -5), (8, 128, 1 << 25, -1), (8, 128, (1 << 25) - 8, -5),
    (1, 64, 1 << 29, -1), (1, 64, (1 << 29) - 128, -5), (3, 64, 178956971, -1),
])
def test_cache_rows(heads, dim, n, code):
    c = ctypes.byref(cache(heads=heads, head_dim=dim))
    wide = heads * dim
    text = "grid" if code == -1 else None
    refused("pk_gpu_kv_write_dev", c, pk.F32, P, wide, P, wide, P, n, None, code=code, text=text)
    refused("pk_gpu_kv_read_dev", c, pk.BF16, P, n, P, wide, P, wide, None, code=code, text=text)


@pytest.mark.parametrize("kv,group,B,code", [(1, 16, 1 << 23, -1), (1, 16, (1 << 23) - 1, -5), (8, 1, 1 << 20, -1),
                                             (1, 40, 2796203, -1), (1, 40, 2796202, -5)])
def test_sequences(kv, group, B, code):
    c = cache(heads=kv)
    wide = kv * group * 128
    attention(c=ctypes.byref(c), heads=kv * group, ldq=wide, ldo=wide, B=B, code=code,
              text="grid" if code == -1 else None)
    if code == -1:
        assert query(c, B, kv * group, 1000, 0) == 0


@pytest.mark.parametrize("K,N,code", [(128, 1 << 29, -1), (128, (1 << 29) - 32, -5), (1, 1 << 30, -1),
                                      (131071, 1 << 20, -1), (131071, (1 << 19) - 16, -5)])
def test_panels(K, N, code):
    assert (pk.load().pk_gpu_w8_panel_bytes(K, N) == 0) == (code == -1)
    refused("pk_gpu_w8_panel_dev", K, N, P, N, P, None, code=code, text="grid" if code == -1 else None)


@pytest.mark.parametrize("M,N,code", [
    (1, 1 << 26, -1), (16, (1 << 26) - 15, -1), (1, (1 << 26) - 16, -5), (17, 1 << 26, -5), (1 << 30, 1, -5),
    (1 << 20, 1 << 19, -1), ((1 << 20) - 256, 1 << 19, -5), (1 << 30, 1 << 30, -1), (0, 1 << 30, -5),
])
def test_products(M, N, code):
    gemm(M=M, N=N, ldr=N, ldc=N, code=code, text="grid" if code == -1 else None)
