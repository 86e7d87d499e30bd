"""CPU: sizes the decoder operators take: workspaces that are large enough for every
smaller call, and launches that would pass the device's limits, refused before
any device is touched.

Pointers here are small aligned numbers that nothing may dereference."""
import ctypes
import re

import pytest

from pkgpu import gpu_available, pk
from test_decode_refusals import P, cache

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
