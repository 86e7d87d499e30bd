"""GPU: attention of one new token per sequence over a 4-bit cache, against the plain
64-bit form within decode_oracle.attention_bound: elements are exact in the matrix
cores' type with their unit, so the bound is that of a 16-bit cache."""
import math

import numpy as np
import pytest

import decode_oracle as do
import more_oracle as mo
from pkgpu import pk
from test_gpu_paged_attention import EDGES, Call, queries, tables

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


CASES = [
    # rows, kv heads, group, dim, page, lengths, max_len, window
    ("f32", 8, 1, 128, 16, [417], 417, 0),
    ("bf16", 2, 4, 128, 32, EDGES, 160, 0),
    ("f16", 1, 5, 64, 16, EDGES, 200, 0),
    ("f32", 3, 2, 256, 64, [300, 1, 0, 77], 300, 0),
    ("f16", 1, 16, 256, 128, [700, 513, 31], 700, 100),
    ("bf16", 2, 17, 64, 16, [129, 64, 5], 129, 0),
    ("f32", 1, 3, 64, 256, [1100, 255, 256, 257], 1100, 0),
    ("f16", 2, 4, 128, 64, [1, 2000, 999], 2000, 33),
    ("bf16", 2, 8, 256, 32, EDGES, 160, 33),
    ("bf16", 1, 2, 128, 16, [30000], 30000, 0),
    ("f32", 1, 2, 128, 16, [9000, 1], 9000, 8000),
]


@pytest.mark.parametrize("rows,kv,group,dim,page,lens,max_len,window", CASES)
def test_against_plain_form(rows, kv, group, dim, page, lens, max_len, window):
    rng = np.random.default_rng(dim * group + max_len)
    B, per = len(lens), (max_len + page - 1) // page
    cache = mo.Cache4(B * per + 1, kv, page, dim, seed=page)
    table = tables(rng, cache, B, per)
    for b, n in enumerate(lens):                      # entries nothing may read
        table[b, (n + page - 1) // page:] = 1 << 30
    q = queries(rng, B, kv * group, dim, rows)
    Call(cache, q, rows, table, lens, max_len, 1.0 / math.sqrt(dim), window, pad=64).check(q, table, lens)
    assert cache.guards_whole()


@pytest.mark.parametrize("rows", ["f32", "f16", "bf16"])
def test_masked_places_may_hold_anything(rows):
    """NaN units and unlike codes in tokens that take no part; absent pages in the middle."""
    import torch
    rng = np.random.default_rng(4)
    B, kv, group, dim, page, most = 4, 2, 2, 128, 16, 250
    per = (most + page - 1) // page
    cache = mo.Cache4(B * per + 2, kv, page, dim, seed=5)
    table = np.arange(B * per, dtype=np.int32).reshape(B, per)
    lens, window = [250, 70, 33, 9], 64
    table[0, 13] = -1
    table[1, 2] = cache.pages
    table[2] = -7
    clean = {n: cache.part(n).clone() for n in cache.arrays}
    seen = np.zeros((cache.pages, page), bool)
    for b, n in enumerate(lens):
        for t in range(max(0, n - window), n):
            if 0 <= table[b, t // page] < cache.pages:
                seen[table[b, t // page], t % page] = True
    hide = torch.from_numpy(~seen).to("cuda:0")[:, None, :, None]
    for name in cache.arrays:
        p = cache.part(name)
        p.copy_(torch.where(hide, torch.full_like(p, 255), p))
    q = queries(rng, B, kv * group, dim, rows)
    c = Call(cache, q, rows, table, lens, most, 0.09, window)
    got = c.run()
    assert np.isfinite(got).all() and np.all(got[2] == 0)
    for n, t in clean.items():
        cache.part(n).copy_(t)
    c.check(q, table, lens)
    assert np.array_equal(do.values(c.out)[:B, :c.wide].reshape(got.shape), got)


def test_a_nan_group_that_is_seen():
    """A value's NaN group makes its 32 elements NaN, a key's the whole head."""
    rng = np.random.default_rng(8)
    cache = mo.Cache4(2, 2, 16, 64, seed=5)
    cache.part("v_scale")[0, 1, 3, 1] = 255
    cache.part("k_scale")[1, 0, 2, 0] = 255
    q = queries(rng, 1, 4, 64, "bf16")
    got = Call(cache, q, "bf16", np.array([[0, 1]], np.int32), [20], 20, 0.125, 0).run()
    assert np.isnan(got[0, :2]).all() and np.isnan(got[0, 2:, 32:]).all() and np.isfinite(got[0, 2:, :32]).all()


@pytest.mark.parametrize("rows,dim", [("bf16", 128), ("f32", 64), ("f32", 256)])
def test_values_near_the_largest_float(rows, dim):
    """Units of 2^125, 6 of which is 2.55e38: outputs are means of such values (weights 2^-18 off, as for the
    largest values of other caches)."""
    rng = np.random.default_rng(dim)
    page, kv, group, lens, max_len = 16, 1, 2, [700, 33], 700
    B, per = 2, (700 + 15) // 16
    cache = mo.Cache4(B * per, kv, page, dim, seed=1)
    table = np.arange(B * per, dtype=np.int32).reshape(B, per)
    v = cache.part("v")
    v.copy_((v & 0x07) | 0x70)                     # positive, every other one 6
    cache.part("v_scale").fill_(252)
    q = queries(rng, B, kv * group, dim, rows)
    for scale in (1.0 / math.sqrt(dim), 0.0):
        c = Call(cache, q, rows, table, lens, max_len, scale, 0)
        got = c.run()
        want, _, a, s, xx = do.attention(cache, q, table, lens, max_len, scale, 0)
        tol = do.attention_bound(want, a, s, xx, max(lens), dim, "e2m1", rows) + 2.0 ** -18 * a
        assert np.all(np.abs(got - want) <= tol), float(np.nanmax(np.abs(got - want) / tol))


def test_a_step_writes_then_attends():
    """40 steps of write + attend from an empty 4-bit cache."""
    import torch
    rng = np.random.default_rng(13)
    B, kv, group, dim, page, steps = 3, 2, 2, 64, 16, 40
    per = (steps + page - 1) // page
    cache = mo.Cache4(B * per, kv, page, dim, filled=False)
    table = tables(rng, cache, B, per)
    for t in range(steps):
        kvrow = torch.from_numpy(rng.normal(0, 1, (B, 2 * kv * dim)).astype(np.float32)).to("cuda:0")
        slots = torch.from_numpy((table[:, t // page] * page + t % page).astype(np.int32)).to("cuda:0")
        pk.call("pk_gpu_kv_write_dev", do.ref(cache.struct()), pk.F32, kvrow.data_ptr(), 2 * kv * dim,
                kvrow.data_ptr() + 4 * kv * dim, 2 * kv * dim, slots.data_ptr(), B, do.stream())
        if t in (0, 1, 15, 16, 31, 39):
            lens = [t + 1] * B
            q = queries(rng, B, kv * group, dim, "f32")
            Call(cache, q, "f32", table, lens, steps, 0.125, 0).check(q, table, lens)
