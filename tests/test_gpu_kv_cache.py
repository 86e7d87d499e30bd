"""GPU: writing a paged key-value cache and reading it back against the plain
64-bit form.

Codes and scales are compared bit for bit with the documented fp32 formula
(one division a row, one product an element, one rounding), and what they
stand for with the rows themselves within half a code's step."""
import numpy as np
import pytest

import decode_oracle as do
from pkgpu import pk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


def rows_of(rng, n, wide, ld, kind):
    import torch
    x = rng.normal(0, 1, (n, ld)).astype(np.float32)
    x[:, rng.integers(0, wide, max(1, wide // 64))] *= 8
    return torch.from_numpy(x).to(do.torch_type(kind)).to("cuda:0")


def distinct_slots(rng, n, pages, page):
    return rng.permutation(pages * page)[:n].astype(np.int32)


def write(cache, kind, k, ldk, v, ldv, slots):
    import torch
    d = torch.from_numpy(np.asarray(slots, np.int32)).to("cuda:0")
    pk.call("pk_gpu_kv_write_dev", do.ref(cache.struct()), do.FLOATS[kind], k.data_ptr(), ldk, v.data_ptr(), ldv,
            d.data_ptr(), len(slots), do.stream())
    torch.cuda.synchronize()


def read(cache, kind, slots, fill=7.0, ld=None):
    import torch
    wide = cache.heads * cache.dim
    ld = ld or wide
    out = [torch.full((len(slots), ld), fill, dtype=do.torch_type(kind), device="cuda:0") for _ in range(2)]
    d = torch.from_numpy(np.asarray(slots, np.int32)).to("cuda:0")
    pk.call("pk_gpu_kv_read_dev", do.ref(cache.struct()), do.FLOATS[kind], d.data_ptr(), len(slots),
            out[0].data_ptr(), ld, out[1].data_ptr(), ld, do.stream())
    torch.cuda.synchronize()
    return out


CASES = [
    # cache, rows, heads, dim, page, n
    ("int8", "f32", 8, 128, 16, 1), ("int8", "bf16", 3, 64, 16, 37), ("int8", "f16", 1, 256, 64, 130),
    ("e4m3", "f32", 2, 128, 32, 65), ("e4m3", "bf16", 8, 128, 256, 300), ("e4m3", "f16", 5, 64, 16, 1),
    ("bf16", "f32", 2, 256, 16, 33), ("bf16", "bf16", 4, 128, 32, 77), ("bf16", "f16", 1, 64, 16, 9),
    ("f16", "f32", 3, 128, 16, 18), ("f16", "f16", 8, 64, 64, 129), ("f16", "bf16", 2, 256, 16, 5),
]


@pytest.mark.parametrize("kind,rows,heads,dim,page,n", CASES)
def test_write_then_read(kind, rows, heads, dim, page, n):
    rng = np.random.default_rng(n * 7 + dim)
    pages = (n + page - 1) // page + 2
    cache = do.Cache(kind, pages, heads, page, dim, seed=n)
    before = {name: do.values(cache.part(name)) for name in cache.arrays}
    wide, ldk, ldv = heads * dim, heads * dim + 64, 2 * heads * dim
    k, v = rows_of(rng, n, wide, ldk, rows), rows_of(rng, n, wide, ldv, rows)
    slots = distinct_slots(rng, n, pages, page)
    if n > 3:
        slots[1], slots[3] = -1, pages * page           # padding: below and past the cache
    write(cache, rows, k, ldk, v, ldv, slots)
    assert cache.guards_whole()
    there = (slots >= 0) & (slots < pages * page)
    for name, x in (("k", k), ("v", v)):
        x = do.values(x)[:, :wide].reshape(n, heads, dim)[there]
        got = do.values(cache.part(name)).transpose(0, 2, 1, 3).reshape(-1, heads, dim)
        rest = np.ones(pages * page, bool)
        rest[slots[there]] = False
        was = before[name].transpose(0, 2, 1, 3).reshape(-1, heads, dim)
        assert np.array_equal(got[rest], was[rest])      # no other slot is touched
        got = got[slots[there]]
        if kind in do.TOP:
            want, scale = do.codes(x, kind)
            sc = do.values(cache.part(name + "_scale")).transpose(0, 2, 1).reshape(-1, heads)
            assert np.array_equal(got, want.astype(np.float64))
            assert np.array_equal(sc[slots[there]], scale.astype(np.float64))
            was = before[name + "_scale"].transpose(0, 2, 1).reshape(-1, heads)
            assert np.array_equal(sc[rest], was[rest])
            assert np.all(np.abs(got * scale[..., None].astype(np.float64) - x) <= do.code_bound(x, kind))
        else:
            assert np.array_equal(got, do.rounded(x, kind).astype(np.float64))
    # back: the same slots in another order, one of them twice, padding left alone
    order = rng.permutation(n)
    again = np.concatenate([slots[order], slots[:1], [-1]]).astype(np.int32)
    back = read(cache, rows, again, ld=wide + 16)
    for name, y in zip(("k", "v"), back):
        stands = cache.rows(name)
        y = do.values(y)
        assert np.all(y[:, wide:] == 7.0)
        for i, s in enumerate(again):
            if not 0 <= s < pages * page:
                assert np.all(y[i] == 7.0)
                continue
            want = do.rounded(stands[s].reshape(-1), rows)
            assert np.array_equal(y[i, :wide], want.astype(np.float64)), (name, i)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_rows_without_a_scale(kind):
    """Zeros, rows below 2^-100, the type's extremes, infinities and NaN."""
    import torch
    heads, dim, page, n = 1, 128, 16, 9
    x = np.random.default_rng(3).normal(0, 1, (n, dim)).astype(np.float32)
    x[0] = 0
    x[1] *= np.float32(2.0 ** -110)
    x[2, 5] = np.inf
    x[3, 9] = np.nan
    x[4, 0] = -np.inf
    x[4, 1] = np.nan
    x[5, 77] = np.finfo(np.float32).max
    x[6, 0] = np.finfo(np.float32).min
    x[7] *= np.float32(2.0 ** -99)
    cache = do.Cache(kind, 2, heads, page, dim, seed=1)
    t = torch.from_numpy(x).to("cuda:0")
    slots = np.arange(n, dtype=np.int32) + 4
    write(cache, "f32", t, dim, t, dim, slots)
    back = [do.values(y) for y in read(cache, "f32", slots)]
    want, scale = do.codes(x, kind)
    for y in back:
        assert np.array_equal(y, want.astype(np.float64) * scale[:, None].astype(np.float64), equal_nan=True) or \
            np.array_equal(y, (want * scale[:, None]).astype(np.float64), equal_nan=True)
        assert np.all(y[0] == 0) and np.all(y[1] == 0)
        assert np.isnan(y[2:5]).all() and np.isfinite(y[5:]).all()


def test_no_rows_is_no_work():
    cache = do.Cache("int8", 1, 1, 16, 64)
    before = cache.rows("k")
    pk.call("pk_gpu_kv_write_dev", do.ref(cache.struct()), pk.F32, None, 64, None, 64, None, 0, do.stream())
    pk.call("pk_gpu_kv_read_dev", do.ref(cache.struct()), pk.F32, None, 0, None, 64, None, 64, do.stream())
    assert np.array_equal(cache.rows("k"), before)


def test_every_slot_of_a_cache_past_4_gib():
    """Element offsets beyond 32 bits: the first, a middle and the last slot of 4.5 GiB of keys."""
    import torch
    heads, dim, page = 8, 256, 256
    pages = (9 << 29) // (heads * dim * page)
    k = torch.zeros((pages * heads * page * dim,), dtype=torch.int8, device="cuda:0")
    v = torch.zeros_like(k)
    ks = torch.zeros((pages * heads * page,), device="cuda:0")
    vs = torch.zeros_like(ks)
    c = pk.KvCache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pk.I8, pages, page, heads, dim)
    last = pages * page - 1
    slots = torch.tensor([0, last, last // 2 + 3], dtype=torch.int32, device="cuda:0")
    x = torch.randn((3, heads * dim), device="cuda:0")
    y = torch.randn((3, heads * dim), device="cuda:0")
    pk.call("pk_gpu_kv_write_dev", do.ref(c), pk.F32, x.data_ptr(), heads * dim, y.data_ptr(), heads * dim,
            slots.data_ptr(), 3, do.stream())
    a, b = torch.empty_like(x), torch.empty_like(x)
    pk.call("pk_gpu_kv_read_dev", do.ref(c), pk.F32, slots.data_ptr(), 3, a.data_ptr(), heads * dim,
            b.data_ptr(), heads * dim, do.stream())
    torch.cuda.synchronize()
    for got, src in ((a, x), (b, y)):
        src = do.values(src).reshape(3, heads, dim)
        assert np.all(np.abs(do.values(got).reshape(3, heads, dim) - src) <= do.code_bound(src, "int8") +
                      2.0 ** -24 * np.abs(src).max())
    tail = k.view(pages, heads, page, dim)[-1, :, -1]
    assert bool((tail.abs().amax(-1) == 127).all())


def test_captured_write_and_read_replay():
    """A graph of both, replayed with new rows between eager work on another stream."""
    import torch
    heads, dim, page, n = 4, 128, 16, 21
    cache = do.Cache("int8", 4, heads, page, dim, filled=False)
    st = cache.struct()
    wide = heads * dim
    x = torch.zeros((n, wide), device="cuda:0")
    out = [torch.zeros_like(x) for _ in range(2)]
    slots = torch.from_numpy(distinct_slots(np.random.default_rng(0), n, 4, page)).to("cuda:0")
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        pk.call("pk_gpu_kv_write_dev", do.ref(st), pk.F32, x.data_ptr(), wide, x.data_ptr(), wide, slots.data_ptr(),
                n, s.cuda_stream)
        pk.call("pk_gpu_kv_read_dev", do.ref(st), pk.F32, slots.data_ptr(), n, out[0].data_ptr(), wide,
                out[1].data_ptr(), wide, s.cuda_stream)
    for i in range(3):
        new = torch.randn((n, wide), device="cuda:0")
        x.copy_(new)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        src = do.values(new).reshape(n, heads, dim)
        for y in out:
            err = np.abs(do.values(y).reshape(n, heads, dim) - src)
            assert np.all(err <= do.code_bound(src, "int8") + 2.0 ** -24 * np.abs(src).max())
