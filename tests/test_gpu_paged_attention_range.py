"""GPU: paged attention at the ends of its types' ranges, and the bits that its
softmax weights keep, against the plain 64-bit form."""
import math

import numpy as np
import pytest

import decode_oracle as do
from pkgpu import pk
from test_gpu_paged_attention import Call, queries, tables

pytestmark = pytest.mark.gpu

LARGE = 3.3e38          # within the largest float, 3.4028e38, and the largest bf16, 3.3895e38


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


@pytest.mark.parametrize("signs", [False, True])
@pytest.mark.parametrize("kind,rows,kv,group,dim,lens,max_len", [
    ("int8", "f32", 2, 3, 128, [700, 33, 40], 700), ("int8", "bf16", 1, 2, 64, [3000, 1, 500], 3000),
    ("e4m3", "bf16", 2, 1, 256, [600, 20, 31], 600), ("e4m3", "f32", 1, 2, 256, [2000, 64, 31], 2000),
    ("bf16", "bf16", 2, 4, 128, [700, 17, 300], 700), ("bf16", "f32", 1, 2, 64, [5000, 2, 900], 5000),
    ("bf16", "f32", 1, 1, 256, [900, 256, 9], 900),
])
def test_values_near_the_largest_float(kind, rows, kv, group, dim, lens, max_len, signs):
    """Values of up to 3.3e38: outputs are means of them, so they stay finite.  The last sequence's are ordinary.

    To be formed within the range, weights may be scaled by 2^-40 or so: a weight's
    exponent then is a number below 64, half of whose last place is 2^-19; that enters the weight and the
    weights' sum, ln 2 of it each: 2^-18 of a more than attention_bound."""
    import torch
    rng = np.random.default_rng(dim + max_len)
    page, B = 16, len(lens)
    per = (max_len + page - 1) // page
    cache = do.Cache(kind, B * per, kv, page, dim, seed=1)
    table = np.arange(B * per, dtype=np.int32).reshape(B, per)
    v = cache.part("v")
    big = v[:(B - 1) * per]
    size = torch.from_numpy(rng.uniform(0.2, 1.0, tuple(big.shape)).astype(np.float32)).to("cuda:0")
    if signs:
        size = size * torch.from_numpy(rng.choice([-1.0, 1.0], tuple(big.shape)).astype(np.float32)).to("cuda:0")
    top = do.TOP.get(kind, LARGE)
    x = size * top
    x = (x.round() if kind == "int8" else x).to(big.dtype)
    big.view(torch.uint8).copy_(x.view(torch.uint8))
    if kind in do.TOP:
        cache.part("v_scale")[:(B - 1) * per] = LARGE / top
    q = queries(rng, B, kv * group, dim, rows)
    for scale in (1.0 / math.sqrt(dim), 0.0, 1.0):
        c = Call(cache, q, rows, table, lens, max_len, scale, 0)
        got = c.run()
        want, lse, a, s, xx = do.attention(cache, q, table, lens, max_len, scale, 0)
        n = max(lens)
        tol = do.attention_bound(want, a, s, xx, n, dim, kind, rows) + 2.0 ** -18 * a
        err = np.abs(got - want)
        assert np.all(err <= tol), (scale, float(np.nanmax(err / tol)), np.argwhere(~(err <= tol))[:4].tolist())
        d = (dim + 8) * 2.0 ** -23 * xx + 6 * 2.0 ** -24 * s + 2.0 ** -18
        ltol = d + (n / 16 + 72) * 2.0 ** -23 + 4 * 2.0 ** -24 * np.abs(lse)
        assert np.all(np.abs(do.values(c.lse)[:B] - lse) <= ltol)


def test_values_that_grow_along_a_sequence():
    """Ordinary values in the first tiles of each wave, the largest behind them, and scores that keep rising."""
    import torch
    rng = np.random.default_rng(2)
    page, n, dim = 16, 1800, 64
    per = (n + page - 1) // page
    cache = do.Cache("bf16", per, 1, page, dim, seed=1)
    table = np.arange(per, dtype=np.int32)[None]
    cache.part("v")[per // 2:] = torch.from_numpy(rng.uniform(0.5, 1.0, (per - per // 2, 1, page, dim)).astype(np.float32)
                                                  * np.float32(LARGE)).to(torch.bfloat16).to("cuda:0")
    k = cache.part("k")
    k.zero_()
    k[:, 0, :, 0] = torch.linspace(0, 30, per * page, device="cuda:0").reshape(per, page).to(torch.bfloat16)
    q = np.zeros((1, 2, dim))
    q[0, :, 0] = 1.0
    c = Call(cache, q, "f32", table, [n], n, 1.0, 0)
    got = c.run()
    want, _, a, s, x = do.attention(cache, q, table, [n], n, 1.0, 0)
    assert np.all(np.abs(got - want) <= do.attention_bound(want, a, s, x, n, dim, "bf16", "f32") + 2.0 ** -18 * a)


def test_f32_queries_near_the_largest_float():
    """Queries that bf16 would round to infinity, over a bf16 cache with keys small enough for scores of 1 or so."""
    rng = np.random.default_rng(4)
    page, n, dim = 16, 100, 64
    cache = do.Cache("bf16", 7, 2, page, dim, seed=1)
    k = cache.part("k")
    k.copy_((k.float() * 2.0 ** -60).to(k.dtype))
    table = np.arange(7, dtype=np.int32)[None]
    q = rng.choice([-1.0, 1.0], (1, 4, dim)) * np.float32(3.4e38).astype(np.float64)
    Call(cache, q, "f32", table, [n], n, 2.0 ** -71, 0).check(q, table, [n])


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_weights_over_f16_caches_keep_22_bits(dim):
    """Two f16 terms of a weight: half a step of the second relative to the weight is 2^-22, where a second
    term is below f16's normal range 2^-25, which is 2^-32 of the maximum's weight, 2^7.  Few tokens with flat
    scores and values that cancel: the outputs, and the other roundings, are small beside a weight's 2^-12."""
    rng = np.random.default_rng(dim)
    page, kv, group, lens = 16, 2, 3, [2, 3, 4, 6, 9, 33]
    B, per = len(lens), 3
    cache = do.Cache("f16", B * per, kv, page, dim, seed=3)
    v = cache.part("v")
    v[:, :, 1::2] = -v[:, :, 0::2]
    table = np.arange(B * per, dtype=np.int32).reshape(B, per)
    q = queries(rng, B, kv * group, dim, "f16")
    got = Call(cache, q, "f16", table, lens, 48, 0.25 / dim, 0).run()
    want, _, a, s, x = do.attention(cache, q, table, lens, 48, 0.25 / dim, 0)
    for b, n in enumerate(lens):
        tol = (do.attention_bound(want[b], a[b], s[b], x[b], n, dim, "f16", "f16")
               - (2.0 ** -11 - 2.0 ** -22) * 1.01 * a[b])
        err = np.abs(got[b] - want[b])
        assert np.all(err <= tol), (n, float((err / tol).max()), int((err > tol).sum()))


@pytest.mark.parametrize("kind,rows,dim,n", [("f16", "f16", 128, 100), ("f16", "f16", 256, 1500), ("bf16", "bf16", 64, 700),
                                             ("bf16", "bf16", 256, 60), ("bf16", "f32", 128, 100), ("bf16", "f32", 64, 3000)])
def test_infinite_values_that_are_seen(kind, rows, dim, n):
    """A mean over an infinite value is that infinity, over both infinities or a NaN it is NaN, and the other
    elements of the head are what they are without it (weights 2^-18 off, as for the largest values)."""
    rng = np.random.default_rng(dim)
    page, kv, group = 16, 2, 3
    per = (n + page - 1) // page
    cache = do.Cache(kind, per, kv, page, dim, seed=4)
    table = np.arange(per, dtype=np.int32)[None]
    q = queries(rng, 1, kv * group, dim, rows)
    c = Call(cache, q, rows, table, [n], n, 0.05, 0)
    v = cache.part("v")
    v[0, 1, 3, [2, 7, 11, 40]] = 0.0
    v[per - 1, 1, 1, [2, 7, 11, 40]] = 0.0
    want, _, a, s, x = do.attention(cache, q, table, [n], n, 0.05, 0)
    tol = do.attention_bound(want, a, s, x, n, dim, kind, rows) + 2.0 ** -18 * a
    v[0, 1, 3, 2], v[0, 1, 3, 7], v[0, 1, 3, 11], v[per - 1, 1, 1, 11] = (float(t) for t in ("inf", "-inf", "inf", "-inf"))
    v[per - 1, 1, 1, 40] = float("nan")
    got = c.run()
    far = got[0, group:]
    assert np.all(far[:, 2] == np.inf) and np.all(far[:, 7] == -np.inf) and np.isnan(far[:, [11, 40]]).all()
    got[0, group:, [2, 7, 11, 40]] = want[0, group:, [2, 7, 11, 40]]
    assert np.all(np.abs(got - want) <= tol), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("kind,rows", [("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32")])
def test_infinite_keys_that_are_seen(kind, rows):
    """Where a key makes a score -inf its token has no weight, where +inf the outputs are NaN; with queries whose
    second and third terms are zeros."""
    rng = np.random.default_rng(6)
    n, dim, page = 90, 64, 16
    cache = do.Cache(kind, 6, 1, page, dim, seed=4)
    table = np.arange(6, dtype=np.int32)[None]
    q = queries(rng, 1, 3, dim, "bf16" if kind == "bf16" else "f16")
    q[0, :, 5] = [1.0, 0.5, -2.0]
    want, _, a, s, x = do.attention(cache, q, table, [n - 1], n, 0.05, 0)
    cache.part("k")[(n - 1) // page, 0, (n - 1) % page, 5] = -float("inf")
    got = Call(cache, q, rows, table, [n], n, 0.05, 0).run()
    assert np.isnan(got[0, 2]).all()
    tol = do.attention_bound(want, a, s, x, n, dim, kind, rows)
    assert np.all(np.abs(got - want)[0, :2] <= tol[0, :2])
