"""GPU: paged attention whose sequences are split over several workgroups, against the
plain 64-bit form within the bound of decode_oracle.attention_bound.  Each case
asserts the split it is there for, as the refusal of a missing workspace names it."""
import math
import re

import numpy as np
import pytest

import decode_oracle as do
from pkgpu import pk
from test_gpu_paged_attention import Call, queries, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


def splits(c):
    """Chunks of the longest sequence: what the call itself asks of a workspace, a chunk's share being dim + 2."""
    lib = pk.load()
    rc = lib.pk_gpu_paged_attention_dev(
        do.ref(c.st), do.FLOATS[c.rows], c.q.data_ptr(), c.ld, c.heads, c.table.data_ptr(), c.table.shape[1],
        c.lens.data_ptr(), c.B, c.max_len, c.scale, c.window, c.out.data_ptr(), c.ld, None, None, 0, do.stream())
    assert rc == -1
    need = int(re.search(r"workspace of (\d+) floats", lib.pk_gpu_last_error().decode()).group(1))
    each = c.B * c.heads * (c.cache.dim + 2)
    assert need % each == 0
    return need // each


CASES = [
    # cache, rows, kv heads, group, dim, page, lengths, max_len, window, splits
    # a window over several chunks, each sequence's own first token; the f16 weights' factor in (m, l) and lse
    ("f16", "f16", 2, 4, 128, 32, [6000, 3517], 6000, 3000, 12),
    ("f16", "f16", 1, 3, 256, 16, [2100, 0, 1025, 768], 2100, 0, 9),
    ("bf16", "bf16", 2, 2, 64, 16, [2500, 1031, 1000, 31], 2600, 1001, 5),
    ("int8", "f32", 1, 2, 128, 64, [4999, 1, 257], 5000, 4970, 20),
    # heads of 256 in 4 and in 8 waves, and more chunks than the join asks for at once
    ("e4m3", "f32", 1, 2, 256, 64, [9000], 9000, 0, 36),
    ("int8", "bf16", 1, 4, 256, 32, [8192, 4097], 9000, 0, 36),
    ("bf16", "f32", 1, 1, 256, 16, [5000, 256, 257], 5000, 0, 20),
    # more chunks than a wave of the join has lanes, and as many as it has threads
    ("bf16", "bf16", 1, 2, 64, 16, [40000], 40000, 0, 157),
    ("e4m3", "f16", 1, 1, 64, 256, [130900], 131072, 0, 256),
    # chunks of several rounds
    ("int8", "bf16", 8, 1, 128, 32, [6000, 767, 768, 769], 6000, 0, 8),
    ("bf16", "f32", 4, 1, 64, 16, [3000] + [1024 * (i % 3) + i for i in range(15)], 3000, 2900, 4),
    # several tiles of query heads
    ("int8", "f16", 2, 20, 64, 16, [1500, 900], 1500, 0, 6),
]


@pytest.mark.parametrize("kind,rows,kv,group,dim,page,lens,max_len,window,want", CASES)
def test_against_plain_form(kind, rows, kv, group, dim, page, lens, max_len, window, want):
    rng = np.random.default_rng(dim * group + max_len)
    B, per = len(lens), (max_len + page - 1) // page
    cache = do.Cache(kind, B * per + 1, kv, page, dim, seed=page)
    table = tables(rng, cache, B, per)
    for b, n in enumerate(lens):                      # entries nothing may read
        table[b, (n + page - 1) // page:] = 1 << 30
    table[0, 5] = -1                                  # a page that is absent
    q = queries(rng, B, kv * group, dim, rows)
    c = Call(cache, q, rows, table, lens, max_len, 1.0 / math.sqrt(dim), window)
    assert splits(c) == want
    c.check(q, table, lens)
    assert cache.guards_whole()


def test_the_same_call_gives_the_same_bits():
    """Eight calls with workspaces that held other things."""
    import torch
    rng = np.random.default_rng(3)
    B, kv, dim, page, most = 3, 2, 128, 16, 5000
    per = (most + page - 1) // page
    cache = do.Cache("bf16", B * per, kv, page, dim, seed=2)
    table = tables(rng, cache, B, per)
    q = queries(rng, B, 4 * kv, dim, "bf16")
    c = Call(cache, q, "bf16", table, [most, 2222, 17], most, 0.09, 0)
    first = c.run()
    for i in range(7):
        c.ws[:c.floats] = torch.randn((c.floats,), device="cuda:0") * 10.0 ** (i - 3)
        assert np.array_equal(c.run(), first)
