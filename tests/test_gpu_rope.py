"""GPU: rotary positions of rows and on the way into the cache, against the plain 64-bit
form within the bound of its roundings (more_oracle.turned_bound)."""
import ctypes

import numpy as np
import pytest

import decode_oracle as do
import more_oracle as mo
from pkgpu import pk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


def freqs_of(rot, base=10000.0):
    f = np.zeros(rot // 2, np.float32)
    pk.call("pk_gpu_rope_freqs", rot, base, pk.ROPE_PLAIN, 1.0, 0.0, 0.0, 0.0, f.ctypes.data)
    return f


class Rows:
    """Rows at any offset and pitch in a buffer of ones, and the rope over them."""

    def __init__(self, rng, n, heads, dim, rot, interleaved, rows, pad=0, offset=0, scale=1.0, far=5000):
        import torch
        self.n, self.heads, self.dim, self.rot, self.inter, self.rows, self.scale = n, heads, dim, rot, interleaved, rows, scale
        self.wide, self.ld, self.offset = heads * dim, heads * dim + pad, offset
        self.x = do.rounded(rng.normal(0, 2, (n, self.wide)), rows)
        self.pos = rng.integers(-far, far, n).astype(np.int32)
        self.f = freqs_of(rot)
        self.d_f, self.d_pos = (torch.from_numpy(a).to("cuda:0") for a in (self.f, self.pos))
        self.dx = self.buffer()
        self.view(self.dx)[:, :self.wide] = torch.from_numpy(self.x).to(do.torch_type(rows)).to("cuda:0")
        self.rope = pk.Rope(self.d_f.data_ptr(), scale, rot, int(interleaved))

    def buffer(self):
        import torch
        return torch.ones((self.offset + self.n * self.ld + 64,), dtype=do.torch_type(self.rows), device="cuda:0")

    def view(self, b):
        return b[self.offset:self.offset + self.n * self.ld].view(self.n, self.ld)

    def at(self, b):
        return b.data_ptr() + self.offset * b.element_size()

    def want(self):
        return mo.turned(self.x.reshape(self.n, self.heads, self.dim), self.pos, self.f, self.scale, self.rot, self.inter)

    def enqueue(self, y, stream):
        pk.call("pk_gpu_rope_dev", ctypes.byref(self.rope), do.FLOATS[self.rows], self.at(self.dx), self.ld, self.heads,
                self.dim, self.d_pos.data_ptr(), self.n, self.at(y), self.ld, stream)

    def check(self, y):
        got = do.values(self.view(y))
        want, size = self.want()
        tol = mo.turned_bound(want, size, self.rows, 1.0 + np.abs(self.pos.astype(np.float64)).max())
        err = np.abs(got[:, :self.wide].reshape(want.shape) - want)
        assert np.all(err <= tol), (float((err / tol).max()), np.argwhere(err > tol)[:4].tolist())
        stays = got[:, :self.wide].reshape(want.shape)[..., self.rot:]
        assert np.array_equal(stays, want[..., self.rot:])                   # to the bit
        # nothing between rows, before the first or behind the last is touched
        assert np.all(got[:, self.wide:] == 1) and bool((y[:self.offset] == 1).all()) and bool((y[-64:] == 1).all())


CASES = [
    # rows, n, heads, dim, rot, interleaved, pad, offset
    ("f32", 33, 8, 128, 128, False, 0, 0), ("bf16", 1, 32, 128, 128, True, 64, 0), ("f16", 37, 3, 64, 64, False, 8, 8),
    ("bf16", 5, 2, 256, 64, False, 0, 0), ("f32", 7, 5, 128, 96, True, 4, 4), ("f16", 9, 1, 128, 48, False, 0, 0),
    ("bf16", 3000, 2, 64, 64, True, 0, 0), ("f32", 2049, 3, 64, 32, False, 0, 0),
    # one element at a time: odd pitches and offsets, turning parts that are no whole pieces
    ("bf16", 11, 3, 128, 128, False, 3, 1), ("f16", 11, 3, 64, 26, True, 0, 0), ("f32", 11, 3, 128, 24, False, 1, 3),
    ("f32", 4, 2, 2, 2, True, 0, 0), ("bf16", 4, 3, 6, 4, False, 0, 0), ("f32", 3, 1, 1024, 1024, False, 0, 0),
    ("bf16", 2100, 1, 1024, 1022, True, 1, 0), ("f16", 6, 7, 33, 32, False, 0, 0), ("f32", 2, 300, 4, 2, False, 0, 0),
]


@pytest.mark.parametrize("rows,n,heads,dim,rot,interleaved,pad,offset", CASES)
@pytest.mark.parametrize("in_place", [False, True])
def test_rows(rows, n, heads, dim, rot, interleaved, pad, offset, in_place):
    import torch
    r = Rows(np.random.default_rng(n + dim), n, heads, dim, rot, interleaved, rows, pad, offset, scale=1.0 if pad else 1.25)
    y = r.dx if in_place else r.buffer()
    r.enqueue(y, do.stream())
    torch.cuda.synchronize()
    r.check(y)


def test_far_positions():
    """Angles of 2^31: the product of position and frequency is rounded to 2^-22 there at most."""
    import torch
    r = Rows(np.random.default_rng(1), 8, 2, 64, 64, False, "f32")
    r.pos[:] = [2 ** 31 - 1, -2 ** 31, 2 ** 31 - 5, 2 ** 24 + 1, 1 << 30, -(1 << 30) + 1, 0, 1]
    r.d_pos.copy_(torch.from_numpy(r.pos))
    y = r.buffer()
    r.enqueue(y, do.stream())
    torch.cuda.synchronize()
    # numpy's own product is off by as much
    want, size = r.want()
    err = np.abs(do.values(r.view(y)).reshape(want.shape) - want)
    assert np.all(err <= mo.turned_bound(want, size, "f32", 2.0 ** 32))


def test_there_and_back():
    """Turned by p and by -p, a row is what it was, within two turns' roundings."""
    import torch
    r = Rows(np.random.default_rng(2), 50, 4, 128, 96, True, "f32")
    y = r.buffer()
    r.enqueue(y, do.stream())
    r.d_pos.neg_()
    r.dx.copy_(y)
    r.enqueue(y, do.stream())
    torch.cuda.synchronize()
    x = r.x.reshape(50, 4, 128).astype(np.float64)
    _, size = r.want()
    err = np.abs(do.values(r.view(y)).reshape(x.shape) - x)
    assert np.all(err <= 3 * mo.turned_bound(x, size, "f32", 5001.0) + 2.0 ** -23 * size)


def test_nothing_to_do():
    f = np.zeros(4, np.float32)
    r = pk.Rope(f.ctypes.data, 1.0, 8, 0)
    pk.call("pk_gpu_rope_dev", ctypes.byref(r), pk.F32, None, 8, 1, 8, None, 0, None, 8, do.stream())
    pk.call("pk_gpu_rope_dev", ctypes.byref(r), pk.F32, None, 8, 0, 8, None, 5, None, 8, do.stream())


def kv_bound(want, size, kind, rows, far):
    """How far what the cache holds may be from the turned keys: the turn's roundings move a row's or group's
    largest value, which the codes' unit follows, and the values themselves; then half a code's step."""
    turn = size * (6 * 2.0 ** -24 + far * 2.0 ** -53)
    if kind in do.TOP:
        return do.code_bound(want, kind) + 2.1 * turn.max(-1, keepdims=True)
    if kind == "e2m1":        # a unit that the turn's roundings double: half a step of the larger one
        g = np.abs(want).reshape(want.shape[:-1] + (-1, mo.GROUP)).max(-1, keepdims=True)
        u = 2.0 ** np.ceil(np.log2(np.maximum(g, 1e-300) / 7 * (1 + 2.0 ** -20)))
        y = np.abs(want) / np.repeat(u, mo.GROUP, -1).reshape(want.shape) * (1 + 2.0 ** -20)
        step = np.where(y < 2, 0.5, np.where(y < 4, 1.0, 2.0))
        return step / 2 * np.repeat(u, mo.GROUP, -1).reshape(want.shape) + 2 * turn.max(-1, keepdims=True)
    return do.HALF[kind] * np.abs(want) * 1.01 + 1.01 * turn + 2.0 ** -24 * (kind == "f16")


WRITES = [
    # cache, rows, n, query heads, kv heads, dim, page, rot, interleaved
    ("bf16", "bf16", 33, 32, 8, 128, 16, 128, False), ("bf16", "f32", 7, 4, 2, 64, 32, 64, True),
    ("f16", "f16", 129, 5, 5, 256, 16, 128, False), ("f16", "f32", 1, 16, 1, 128, 64, 24, False),
    ("int8", "bf16", 3000, 4, 2, 128, 64, 64, True), ("int8", "f32", 19, 3, 3, 64, 16, 26, False),
    ("e4m3", "f16", 65, 8, 4, 128, 256, 96, True), ("e4m3", "f32", 5, 2, 2, 256, 16, 250, True),
    ("e2m1", "f32", 40, 6, 3, 128, 16, 128, False), ("e2m1", "bf16", 2100, 1, 1, 64, 16, 40, True),
    ("e2m1", "f16", 3, 2, 1, 256, 32, 18, False), ("int8", "bf16", 4, 0, 9, 64, 16, 64, False),
]


@pytest.mark.parametrize("kind,rows,n,heads,kv,dim,page,rot,interleaved", WRITES)
@pytest.mark.parametrize("in_place", [False, True])
def test_into_the_cache(kind, rows, n, heads, kv, dim, page, rot, interleaved, in_place):
    import torch
    rng = np.random.default_rng(n + rot)
    pages = (n + page - 1) // page + 2
    cache = mo.cache_of(kind, pages, kv, page, dim, seed=3)
    before = {m: cache.rows(m) for m in ("k", "v")}
    q = Rows(rng, n, max(heads, 1), dim, rot, interleaved, rows, pad=64, scale=0.75)
    wide, ld = kv * dim, 2 * kv * dim + 64            # keys and values side by side, as a fused projection leaves them
    new = do.rounded(rng.normal(0, 1, (n, ld)), rows)
    d_new = torch.from_numpy(new).to(do.torch_type(rows)).to("cuda:0")
    slots = rng.permutation(pages * page)[:n].astype(np.int32)
    if n > 3:
        slots[1], slots[3] = -1, pages * page
    d_slots = torch.from_numpy(slots).to("cuda:0")
    y = q.dx if in_place else q.buffer()
    es = d_new.element_size()
    pk.call("pk_gpu_rope_kv_write_dev", ctypes.byref(q.rope), do.ref(cache.struct()), do.FLOATS[rows],
            q.at(q.dx) if heads else None, q.ld, heads, q.at(y) if heads else None, q.ld, d_new.data_ptr(), ld,
            d_new.data_ptr() + wide * es, ld, q.d_pos.data_ptr(), d_slots.data_ptr(), n, do.stream())
    torch.cuda.synchronize()
    if heads:
        q.check(y)
    assert cache.guards_whole() and np.array_equal(do.values(d_new), new.astype(np.float64))
    there = (slots >= 0) & (slots < pages * page)
    rest = np.ones(pages * page, bool)
    rest[slots[there]] = False
    k, v = (new[:, i * wide:(i + 1) * wide].reshape(n, kv, dim)[there] for i in range(2))
    want, size = mo.turned(k, q.pos[there], q.f, 0.75, rot, interleaved)
    got = {m: cache.rows(m) for m in ("k", "v")}
    for m in ("k", "v"):
        assert np.array_equal(got[m][rest], before[m][rest])
    tol = kv_bound(want, size, kind, rows, 5001.0)
    err = np.abs(got["k"][slots[there]] - want)
    assert np.all(err <= tol), (float((err / tol).max()), np.argwhere(err > tol)[:4].tolist())
    # values as pk_gpu_kv_write_dev writes them, to the bit
    other = mo.cache_of(kind, pages, kv, page, dim, seed=3)
    pk.call("pk_gpu_kv_write_dev", do.ref(other.struct()), do.FLOATS[rows], d_new.data_ptr(), ld,
            d_new.data_ptr() + wide * es, ld, d_slots.data_ptr(), n, do.stream())
    torch.cuda.synchronize()
    for m in cache.arrays:
        if m[0] == "v":
            assert torch.equal(cache.part(m).view(torch.uint8), other.part(m).view(torch.uint8))


def test_keys_that_do_not_turn_are_written_alike():
    """At position 0 a row is what it was: codes and scales as pk_gpu_kv_write_dev's, values' NaN and infinities too."""
    import torch
    n, kv, dim = 6, 2, 128
    x = torch.randn((n, kv * dim), device="cuda:0")
    x[1, 3], x[2, 140], x[3, :dim] = float("nan"), float("inf"), 0.0
    f = torch.from_numpy(freqs_of(64)).to("cuda:0")
    zero, slots = torch.zeros(n, dtype=torch.int32, device="cuda:0"), torch.arange(n, dtype=torch.int32, device="cuda:0")
    for kind in ("int8", "e4m3", "e2m1", "bf16"):
        a, b = (mo.cache_of(kind, 1, kv, 16, dim, seed=1) for _ in range(2))
        r = pk.Rope(f.data_ptr(), 1.0, 64, 1)
        pk.call("pk_gpu_rope_kv_write_dev", ctypes.byref(r), do.ref(a.struct()), pk.F32, None, 0, 0, None, 0, x.data_ptr(),
                kv * dim, x.data_ptr(), kv * dim, zero.data_ptr(), slots.data_ptr(), n, do.stream())
        pk.call("pk_gpu_kv_write_dev", do.ref(b.struct()), pk.F32, x.data_ptr(), kv * dim, x.data_ptr(), kv * dim,
                slots.data_ptr(), n, do.stream())
        torch.cuda.synchronize()
        for row in (0, 3, 4, 5):                    # in the others 0 times an infinity or a NaN enters the pair
            assert np.array_equal(a.rows("k")[row], b.rows("k")[row], equal_nan=True)
        assert np.array_equal(a.rows("v"), b.rows("v"), equal_nan=True)


def test_captured_and_replayed():
    """A graph of both calls, replayed with new rows, positions and slots."""
    import torch
    rng = np.random.default_rng(5)
    n, heads, kv, dim = 9, 4, 2, 64
    cache = mo.cache_of("int8", 4, kv, 16, dim, filled=False)
    st = cache.struct()
    q = Rows(rng, n, heads, dim, 64, False, "f32")
    y, z = q.buffer(), q.buffer()
    kvr = torch.zeros((n, 2 * kv * dim), device="cuda:0")
    slots = torch.zeros(n, dtype=torch.int32, device="cuda:0")

    def enqueue(stream):
        pk.call("pk_gpu_rope_kv_write_dev", ctypes.byref(q.rope), do.ref(st), pk.F32, q.at(q.dx), q.ld, heads, q.at(y), q.ld,
                kvr.data_ptr(), 2 * kv * dim, kvr.data_ptr() + 4 * kv * dim, 2 * kv * dim, q.d_pos.data_ptr(),
                slots.data_ptr(), n, stream)
        q.enqueue(z, stream)
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        enqueue(s.cuda_stream)
    for i in range(3):
        q.x = rng.normal(0, 1, q.x.shape).astype(np.float32)
        q.view(q.dx)[:, :q.wide] = torch.from_numpy(q.x).to("cuda:0")
        q.pos = rng.integers(0, 3000, n).astype(np.int32)
        q.d_pos.copy_(torch.from_numpy(q.pos))
        new = rng.normal(0, 1, (n, 2 * kv * dim)).astype(np.float32)
        kvr.copy_(torch.from_numpy(new))
        at = rng.permutation(64)[:n].astype(np.int32)
        slots.copy_(torch.from_numpy(at))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        q.check(y)
        q.check(z)
        want, size = mo.turned(new[:, :kv * dim].reshape(n, kv, dim), q.pos, q.f, 1.0, 64, False)
        assert np.all(np.abs(cache.rows("k")[at] - want) <= kv_bound(want, size, "int8", "f32", 5001.0))
