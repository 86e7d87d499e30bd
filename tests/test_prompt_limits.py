"""CPU: the attention with rules refuses sizes whose products pass 64 bits, and takes bounds that are far from what
a call holds.  Pointers here are small aligned numbers that nothing may dereference."""
import ctypes

import pytest

from pkgpu import gpu_available, pk
from test_decode_refusals import P, cache, refused
from test_prompt_refusals import rules

# calls that are not refused end without a device, and only so
pytestmark = pytest.mark.skipif(gpu_available(), reason="makes calls with addresses that nothing may read")

TOP = 2 ** 31 - 1


def call(kv, heads, B, rows, new, code, text, length=128, kind=pk.I8, ws=P):
    c = cache(dtype=kind, heads=kv, head_dim=64, n_pages=8, page_size=16)
    refused("pk_gpu_prompt_attention_dev", ctypes.byref(c), pk.BF16, P, heads * 64, heads, P, 1 << 26, P, P, B, rows, new,
            length, rules(), P, heads * 64, None, ws, 1 << 40, None, code=code, text=text)


@pytest.mark.parametrize("kv", [1, 64])
@pytest.mark.parametrize("heads", [64, 1024, 1 << 24])
@pytest.mark.parametrize("B", [1 << 20, 1 << 26, TOP])
@pytest.mark.parametrize("rows,new", [(TOP, 1 << 30), (1 << 24, 1 << 24), (1 << 27, 1 << 27)])
@pytest.mark.parametrize("length", [128, 1 << 30])
def test_sizes_past_64_bits(kv, heads, B, rows, new, length):
    call(kv, heads, B, rows, new, -1, "grid", length=length)


@pytest.mark.parametrize("B,rows,new", [(1, 1 << 20, 1 << 20), (3, 1 << 20, 1 << 20), (1 << 12, 1 << 20, 1 << 20),
                                        (1 << 12, 1000, 1 << 30), (1 << 12, 1 << 20, 3)])
def test_bounds_far_above_the_rows(B, rows, new):
    """As many tiles as rows fill, however many new tokens one sequence may have."""
    for kv in (1, 8):
        call(kv, 64, B, rows, new, -5, None)
