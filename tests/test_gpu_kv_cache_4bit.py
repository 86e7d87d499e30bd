"""GPU: a key-value cache in 4-bit floats: codes and bytes bit for bit against the
documented rule (every step of it is exact), what they stand for within half a step."""
import numpy as np
import pytest

import decode_oracle as do
import more_oracle as mo
from pkgpu import pk
from test_gpu_kv_cache import distinct_slots, read, rows_of, write

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


CASES = [("f32", 8, 128, 16, 1), ("bf16", 3, 64, 16, 37), ("f16", 1, 256, 64, 130), ("f32", 2, 64, 256, 65),
         ("bf16", 8, 128, 32, 301), ("f16", 5, 128, 16, 1), ("bf16", 1, 256, 16, 33), ("f32", 8, 256, 16, 1500)]


@pytest.mark.parametrize("rows,heads,dim,page,n", CASES)
def test_write_then_read(rows, heads, dim, page, n):
    rng = np.random.default_rng(n * 7 + dim)
    pages = (n + page - 1) // page + 2
    cache = mo.Cache4(pages, heads, page, dim, seed=n)
    before = {name: cache.codes(name) for name in ("k", "v")}
    wide, ldk, ldv = heads * dim, heads * dim + 64, 2 * heads * dim
    k, v = rows_of(rng, n, wide, ldk, rows), rows_of(rng, n, wide, ldv, rows)
    slots = distinct_slots(rng, n, pages, page)
    if n > 3:
        slots[1], slots[3] = -1, pages * page           # padding: below and past the cache
    write(cache, rows, k, ldk, v, ldv, slots)
    assert cache.guards_whole()
    there = (slots >= 0) & (slots < pages * page)
    rest = np.ones(pages * page, bool)
    rest[slots[there]] = False
    for name, x in (("k", k), ("v", v)):
        x = do.values(x)[:, :wide].reshape(n, heads, dim)[there]
        code, byte = cache.codes(name)
        assert np.array_equal(code[rest], before[name][0][rest]) and np.array_equal(byte[rest], before[name][1][rest])
        want, unit = mo.codes4(x)
        assert np.array_equal(byte[slots[there]], unit) and np.array_equal(code[slots[there]], want)
        u = np.repeat(2.0 ** (unit.astype(np.float64) - 127), mo.GROUP, -1)
        y = np.abs(x) / u
        step = np.where(y < 2, 0.5, np.where(y < 4, 1.0, 2.0))           # of the codes on both sides
        assert np.all(np.abs(cache.rows(name)[slots[there]] - x) <= step / 2 * u)
    order = rng.permutation(n)
    again = np.concatenate([slots[order], slots[:1], [-1]]).astype(np.int32)
    back = read(cache, rows, again, ld=wide + 16)
    for name, y in zip(("k", "v"), back):
        stands = cache.rows(name)
        y = do.values(y)
        assert np.all(y[:, wide:] == 7.0)
        for i, s in enumerate(again):
            want = do.rounded(stands[s].reshape(-1), rows) if 0 <= s < pages * page else np.full(wide, 7.0)
            assert np.array_equal(y[i, :wide], want.astype(np.float64)), (name, i)


def test_ties_borders_and_ends_of_the_range():
    import torch
    heads, dim, page = 1, 64, 16
    sizes = np.array([0, .25, .5, .75, 1, 1.25, 1.5, 1.75, 2, 2.5, 3, 3.5, 4, 5, 6], np.float32)
    near = np.concatenate([sizes, np.nextafter(sizes, np.float32(9)), np.nextafter(sizes, np.float32(-1))])
    x = np.zeros((16, dim), np.float32)
    x[0, :32], x[0, 32:] = near[:32], -near[:32]
    x[1, :13] = near[32:]
    x[:2, [31, 63]] = 6.0                                  # the unit is 1
    x[2, :32], x[2, 32:] = 7.0, np.nextafter(np.float32(7), np.float32(8))      # the unit changes behind 7
    x[3, 5], x[3, 40] = np.inf, np.nan                     # a group that has none, each
    x[4, 3] = -np.inf
    x[5, 1], x[5, 33] = np.finfo(np.float32).max, np.finfo(np.float32).min
    x[6, 1], x[6, 33] = 2.0 ** -100, np.nextafter(np.float32(2.0 ** -100), np.float32(0))
    x[7] = 2.0 ** -130
    x[8, :] = np.linspace(-6, 6, dim)
    x[9] = np.float32(1.5) * np.exp2(np.arange(dim) - 40.0)
    x[10, ::2] = -0.0
    cache = mo.Cache4(1, heads, page, dim, seed=1)
    t = torch.from_numpy(x).to("cuda:0")
    slots = np.arange(16, dtype=np.int32)
    write(cache, "f32", t, dim, t, dim, slots)
    code, byte = mo.codes4(x)
    for name, y in zip(("k", "v"), read(cache, "f32", slots)):
        got = cache.codes(name)
        assert np.array_equal(got[1][:, 0], byte)
        fine = np.repeat(byte != 255, mo.GROUP, -1)
        assert np.array_equal(got[0][:, 0][fine] & 7, code[fine] & 7)
        assert np.array_equal(mo.stand_for(got[0][:, 0], byte)[fine], mo.stand_for(code, byte)[fine])
        y = do.values(y)
        assert np.array_equal(y, mo.stand_for(code, byte), equal_nan=True)
        assert np.isnan(y[3]).all() and np.isnan(y[4, :32]).all() and np.isfinite(y[5]).all()
        assert np.all(y[6, 32:] == 0) and np.all(y[7] == 0) and y[6, 1] == 2.0 ** -100


def test_every_slot_of_a_cache_past_4_gib():
    """Element offsets beyond 32 bits: 4.5 GiB of keys in 4 bits, 9 G elements."""
    import torch
    heads, dim, page = 8, 256, 256
    pages = (9 << 29) // (heads * dim // 2 * page)
    k = torch.zeros((pages * heads * page * dim // 2,), dtype=torch.uint8, device="cuda:0")
    v = torch.zeros_like(k)
    ks = torch.zeros((pages * heads * page * dim // 32,), dtype=torch.uint8, device="cuda:0")
    vs = torch.zeros_like(ks)
    c = pk.KvCache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pk.E2M1, pages, page, heads, dim)
    last = pages * page - 1
    slots = torch.tensor([0, last, last // 2 + 3], dtype=torch.int32, device="cuda:0")
    x, y = (torch.randn((3, heads * dim), device="cuda:0") for _ in range(2))
    pk.call("pk_gpu_kv_write_dev", do.ref(c), pk.F32, x.data_ptr(), heads * dim, y.data_ptr(), heads * dim,
            slots.data_ptr(), 3, do.stream())
    a, b = torch.empty_like(x), torch.empty_like(x)
    pk.call("pk_gpu_kv_read_dev", do.ref(c), pk.F32, slots.data_ptr(), 3, a.data_ptr(), heads * dim,
            b.data_ptr(), heads * dim, do.stream())
    torch.cuda.synchronize()
    for got, src in ((a, x), (b, y)):
        assert np.array_equal(do.values(got), mo.stand_for(*mo.codes4(do.values(src))))
    assert int((ks != 0).sum()) == 3 * heads * dim // 32 and bool((ks.view(pages, heads, page, -1)[-1, :, -1] != 0).all())


def test_captured_write_and_read_replay():
    import torch
    heads, dim, page, n = 4, 128, 16, 21
    cache = mo.Cache4(4, heads, page, dim, filled=False)
    st, wide = cache.struct(), heads * dim
    x = torch.zeros((n, wide), device="cuda:0")
    out = [torch.zeros_like(x) for _ in range(2)]
    slots = torch.from_numpy(distinct_slots(np.random.default_rng(0), n, 4, page)).to("cuda:0")
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        pk.call("pk_gpu_kv_write_dev", do.ref(st), pk.F32, x.data_ptr(), wide, x.data_ptr(), wide, slots.data_ptr(),
                n, s.cuda_stream)
        pk.call("pk_gpu_kv_read_dev", do.ref(st), pk.F32, slots.data_ptr(), n, out[0].data_ptr(), wide,
                out[1].data_ptr(), wide, s.cuda_stream)
    for i in range(3):
        x.copy_(torch.randn((n, wide), device="cuda:0") * 10.0 ** i)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = mo.stand_for(*mo.codes4(do.values(x)))
        assert all(np.array_equal(do.values(y), want) for y in out)
