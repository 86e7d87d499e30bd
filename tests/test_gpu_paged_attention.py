"""GPU: attention of one new token per sequence over a paged cache, against the
plain 64-bit form within the bound that its roundings add up to
(decode_oracle.attention_bound)."""
import math

import numpy as np
import pytest

import decode_oracle as do
from pkgpu import pk

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


def tables(rng, cache, B, per):
    """Distinct pages for each sequence while there are enough, then shared ones."""
    ids = np.concatenate([rng.permutation(cache.pages) for _ in range(B * per // cache.pages + 1)])
    return ids[:B * per].reshape(B, per).astype(np.int32)


class Call:
    """Inputs on the device and one call."""

    def __init__(self, cache, q, rows, table, lens, max_len, scale, window, pad=0, lse=True):
        import torch
        self.cache, self.rows, self.max_len, self.scale, self.window = cache, rows, max_len, scale, window
        self.B, self.heads, dim = q.shape
        self.wide = self.heads * dim
        self.ld = self.wide + pad
        tt = do.torch_type(rows)
        self.q = torch.zeros((max(1, self.B), self.ld), dtype=tt, device="cuda:0")
        self.q[:self.B, :self.wide] = torch.from_numpy(q.reshape(self.B, -1)).to(tt).to("cuda:0")
        self.out = torch.full((self.B + 1, self.ld), 5.0, dtype=tt, device="cuda:0")
        self.lse = torch.full((self.B + 1, self.heads), 5.0, device="cuda:0") if lse else None
        self.table = torch.from_numpy(np.ascontiguousarray(table)).to("cuda:0")
        self.lens = torch.from_numpy(np.asarray(lens, np.int32)).to("cuda:0")
        self.st = cache.struct()
        self.floats = pk.load().pk_gpu_paged_attention_ws_floats(do.ref(self.st), self.B, self.heads, max_len, window)
        self.ws = torch.full((self.floats + 64,), float("nan"), device="cuda:0")

    def enqueue(self, stream):
        pk.call("pk_gpu_paged_attention_dev", do.ref(self.st), do.FLOATS[self.rows], self.q.data_ptr(), self.ld,
                self.heads, self.table.data_ptr(), self.table.shape[1], self.lens.data_ptr(), self.B, self.max_len,
                self.scale, self.window, self.out.data_ptr(), self.ld,
                self.lse.data_ptr() if self.lse is not None else None, self.ws.data_ptr(), self.floats, stream)

    def run(self):
        import torch
        self.enqueue(do.stream())
        torch.cuda.synchronize()
        # nothing behind the last row, between rows or behind the workspace is touched
        assert bool((self.out[self.B:] == 5).all()) and bool((self.out[:, self.wide:] == 5).all())
        assert bool(self.ws[self.floats:].isnan().all())
        if self.lse is not None:
            assert bool((self.lse[self.B:] == 5).all())
        return do.values(self.out)[:self.B, :self.wide].reshape(self.B, self.heads, -1)

    def check(self, q, table, lens):
        got = self.run()
        want, lse, a, s, x = do.attention(self.cache, q, table, lens, self.max_len, self.scale, self.window)
        n = max(1, min(self.max_len, max(lens)))
        tol = do.attention_bound(want, a, s, x, n, self.cache.dim, self.cache.kind, self.rows)
        err = np.abs(got - want)
        assert np.all(err <= tol), (float((err - tol).max()), np.argwhere(err > tol)[:4].tolist())
        if self.lse is not None:
            got = do.values(self.lse)[:self.B]
            d = (self.cache.dim + 8) * 2.0 ** -23 * x + 6 * 2.0 ** -24 * s
            ltol = d + (n / 16 + 72) * 2.0 ** -23 + 4 * 2.0 ** -24 * np.where(np.isfinite(lse), np.abs(lse), 0)
            none = np.isneginf(lse)
            assert np.array_equal(np.isneginf(got), none)
            assert np.all(np.abs(got[~none] - lse[~none]) <= ltol[~none])


def queries(rng, B, heads, dim, rows):
    return do.rounded(rng.normal(0, 1, (B, heads, dim)), rows).astype(np.float64)


EDGES = [0, 1, 15, 16, 17, 31, 32, 33, 127, 128, 129, 160]

CASES = [
    # cache, rows, kv heads, group, dim, page, lengths, max_len, window
    ("int8", "f32", 8, 1, 128, 16, [417], 417, 0),
    ("int8", "bf16", 2, 4, 128, 32, EDGES, 160, 0),
    ("int8", "f16", 1, 5, 64, 16, EDGES, 200, 0),
    ("int8", "f32", 3, 2, 256, 64, [300, 1, 0, 77], 300, 0),
    ("e4m3", "f16", 1, 16, 256, 128, [700, 513, 31], 700, 100),
    ("e4m3", "bf16", 2, 17, 64, 16, [129, 64, 5], 129, 0),
    ("e4m3", "f32", 1, 3, 128, 256, [1100, 255, 256, 257], 1100, 0),
    ("bf16", "bf16", 4, 4, 128, 64, [1, 2000, 999], 2000, 0),
    ("bf16", "f32", 2, 2, 64, 16, EDGES, 160, 33),
    ("bf16", "f32", 1, 8, 256, 32, [95, 96, 97], 97, 0),
    ("f16", "f16", 2, 8, 128, 16, EDGES, 160, 0),
    ("f16", "f16", 1, 40, 64, 32, [333], 4096, 1),
    ("f16", "f16", 3, 1, 256, 16, [48, 0, 1], 48, 16),
    ("bf16", "bf16", 1, 1, 64, 4096, [5000], 5000, 0),
]


@pytest.mark.parametrize("kind,rows,kv,group,dim,page,lens,max_len,window", CASES)
def test_against_plain_form(kind, rows, kv, group, dim, page, lens, max_len, window):
    rng = np.random.default_rng(dim * group + max_len)
    B, per = len(lens), (max_len + page - 1) // page
    cache = do.Cache(kind, B * per + 1, kv, page, dim, seed=page)
    table = tables(rng, cache, B, per)
    for b, n in enumerate(lens):                      # entries nothing may read
        table[b, (n + page - 1) // page:] = 1 << 30
    q = queries(rng, B, kv * group, dim, rows)
    Call(cache, q, rows, table, lens, max_len, 1.0 / math.sqrt(dim), window, pad=64).check(q, table, lens)


def test_many_sequences_one_launch():
    """Enough (sequence, head) pairs that chunks are longer than a round, ragged, without lse."""
    rng = np.random.default_rng(9)
    B, kv, dim, page, most = 300, 2, 64, 16, 700
    cache = do.Cache("int8", 400, kv, page, dim, seed=2)
    lens = rng.integers(0, most + 1, B)
    table = tables(rng, cache, B, (most + page - 1) // page)
    q = queries(rng, B, kv, dim, "bf16")
    Call(cache, q, "bf16", table, lens, most, 0.125, 0, lse=False).check(q, table, lens)


@pytest.mark.parametrize("window", [0, 1130])
def test_longest_first(window):
    """More workgroups than run at a time: sequences in order of length, many of them equal,
    lengths out of range among them."""
    rng = np.random.default_rng(19)
    B, kv, dim, page, most = 67, 8, 64, 16, 1200
    cache = do.Cache("e4m3", 500, kv, page, dim, seed=2)
    lens = rng.integers(0, most + 1, B)
    lens[10:30] = 640
    lens[3], lens[5], lens[66] = -4, 1 << 30, most
    table = tables(rng, cache, B, (most + page - 1) // page)
    q = queries(rng, B, kv, dim, "f16")
    Call(cache, q, "f16", table, lens, most, 0.125, window).check(q, table, np.clip(lens, 0, most))


def test_more_pairs_than_chunks():
    """So many pairs that no sequence is split: no workspace."""
    rng = np.random.default_rng(10)
    B, kv, dim, page, most = 1100, 2, 64, 16, 150
    cache = do.Cache("bf16", 300, kv, page, dim, seed=2)
    lens = rng.integers(0, most + 1, B)
    table = tables(rng, cache, B, (most + page - 1) // page)
    q = queries(rng, B, kv, dim, "bf16")
    c = Call(cache, q, "bf16", table, lens, most, 0.125, 0)
    assert c.floats == 0
    c.check(q, table, lens)


@pytest.mark.parametrize("kind,rows", [("int8", "bf16"), ("e4m3", "f32"), ("bf16", "bf16"), ("f16", "f16")])
def test_masked_places_may_hold_anything(kind, rows):
    """NaN and infinities in pages, scales and queries' unseen tokens; absent pages in the middle."""
    import torch
    rng = np.random.default_rng(4)
    B, kv, group, dim, page, most = 4, 2, 2, 128, 16, 250
    per = (most + page - 1) // page
    cache = do.Cache(kind, B * per + 2, kv, page, dim, seed=5)
    table = np.arange(B * per, dtype=np.int32).reshape(B, per)
    lens, window = [250, 70, 33, 9], 64
    table[0, 13] = -1                      # in the window of sequence 0
    table[1, 2] = cache.pages              # one past the last
    table[2] = -7                          # nothing left of sequence 2
    clean = {n: cache.part(n).clone() for n in cache.arrays}
    nan = float("nan")
    seen = np.zeros((cache.pages, page), bool)
    for b, n in enumerate(lens):
        for t in range(max(0, n - window), n):
            if 0 <= table[b, t // page] < cache.pages:
                seen[table[b, t // page], t % page] = True
    hide = torch.from_numpy(~seen).to("cuda:0")[:, None, :]
    for name in cache.arrays:
        p = cache.part(name)
        h = hide if p.dim() == 3 else hide[..., None]
        if p.dtype == torch.int8:
            p.copy_(torch.where(h, torch.full_like(p, -128), p))
        elif kind == "e4m3" and p.dim() == 4:
            bytes_ = p.view(torch.uint8)
            bytes_.copy_(torch.where(h, torch.full_like(bytes_, 0x7F), bytes_))      # e4m3's NaN
        else:
            alt = torch.where(torch.rand(p.shape, device="cuda:0") < 0.5, nan, float("inf")).to(p.dtype)
            p.copy_(torch.where(h, alt, p))
    q = queries(rng, B, kv * group, dim, rows)
    c = Call(cache, q, rows, table, lens, most, 0.09, window)
    got = c.run()
    assert np.isfinite(got).all() and np.all(got[2] == 0)
    for n, t in clean.items():
        cache.part(n).copy_(t)
    c.check(q, table, lens)                # the same values with nothing hidden there
    assert np.array_equal(do.values(c.out)[:B, :c.wide].reshape(got.shape), got)


def test_lengths_out_of_range_are_bounded():
    rng = np.random.default_rng(6)
    cache = do.Cache("int8", 9, 1, 16, 64, seed=5)
    table = np.arange(9, dtype=np.int32).reshape(1, 9).repeat(3, 0)
    lens = [1 << 30, -5, 100]
    q = queries(rng, 3, 2, 64, "f32")
    c = Call(cache, q, "f32", table, lens, 140, 0.125, 0)
    c.check(q, table, [140, 0, 100])


def test_large_and_flat_scores():
    """Scores of several hundred, where one token takes all, and scale 0, where all weigh the same."""
    rng = np.random.default_rng(8)
    cache = do.Cache("bf16", 40, 2, 16, 64, seed=5)
    table = np.arange(40, dtype=np.int32).reshape(1, 40)
    q = queries(rng, 1, 4, 64, "f32")
    for scale in (20.0, -3.0, 0.0):
        Call(cache, q, "f32", table, [639], 640, scale, 0).check(q, table, [639])


def test_a_value_that_is_seen_passes_its_nan_on():
    rng = np.random.default_rng(8)
    cache = do.Cache("bf16", 2, 2, 16, 64, seed=5)
    cache.part("v")[0, 1, 3, 7] = float("nan")
    q = queries(rng, 1, 4, 64, "bf16")
    got = Call(cache, q, "bf16", np.array([[0, 1]], np.int32), [20], 20, 0.125, 0).run()
    assert np.isnan(got[0, 2:, 7]).all() and np.isfinite(np.delete(got, 7, -1)).all()
    assert np.isfinite(got[0, :2]).all()


def test_two_graphs_and_a_second_stream():
    """Two captured calls with workspaces of their own, replayed side by side with changing
    lengths, give what eager calls give, bit for bit."""
    import torch
    rng = np.random.default_rng(12)
    B, kv, group, dim, page, most = 3, 2, 4, 128, 16, 1500
    per = (most + page - 1) // page
    calls, graphs, streams = [], [], []
    for i in range(2):
        cache = do.Cache("int8", B * per, kv, page, dim, seed=20 + i)
        table = tables(rng, cache, B, per)
        q = queries(rng, B, kv * group, dim, "bf16")
        calls.append(Call(cache, q, "bf16", table, [most, 3, 800], most, 0.09, 0))
        s = torch.cuda.Stream()
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            calls[-1].enqueue(s.cuda_stream)
        graphs.append(g)
        streams.append(s)
    for lens in ([most, 3, 800], [0, 1499, 64], [700, 701, 1]):
        want = []
        for c in calls:
            c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
            want.append(c.run())
            c.out[:B].zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c, w in zip(calls, want):
            assert np.array_equal(do.values(c.out)[:B, :c.wide].reshape(w.shape), w)


def test_two_graphs_take_turns_with_one_workspace():
    """Two captured calls that share a workspace, replayed one after the other on one stream in
    changing order, with eager calls in between that share it too."""
    import torch
    rng = np.random.default_rng(15)
    B, kv, group, dim, page = 2, 2, 4, 64, 16
    calls, graphs = [], []
    s = torch.cuda.Stream()
    for i, most in enumerate((1500, 4000)):
        per = (most + page - 1) // page
        cache = do.Cache("e4m3", B * per, kv, page, dim, seed=30 + i)
        table = tables(rng, cache, B, per)
        q = queries(rng, B, kv * group, dim, "f32")
        calls.append(Call(cache, q, "f32", table, [most, 777], most, 0.125, 0))
    floats = max(c.floats for c in calls)
    shared = torch.full((floats + 64,), float("nan"), device="cuda:0")
    want = [c.run() for c in calls]
    for c in calls:
        c.ws = shared
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            c.enqueue(s.cuda_stream)
        graphs.append(g)
    for order in ((0, 1), (1, 0), (1, 1, 0)):
        for c in calls:
            c.out[:B].zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            for i in order:
                graphs[i].replay()
                calls[1 - i].enqueue(s.cuda_stream)
                graphs[i].replay()
        torch.cuda.synchronize()
        for c, w in zip(calls, want):
            assert np.array_equal(do.values(c.out)[:B, :c.wide].reshape(w.shape), w)


def test_a_step_writes_then_attends():
    """The operators as a decoder uses them: 40 steps of write + attend from an empty int8 cache."""
    import torch
    rng = np.random.default_rng(13)
    B, kv, group, dim, page, steps = 3, 2, 2, 64, 16, 40
    per = (steps + page - 1) // page
    cache = do.Cache("int8", B * per, kv, page, dim, filled=False)
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


def test_a_cache_past_4_gib():
    """The last pages of 4.5 GiB of keys and of values: element offsets beyond 32 bits."""
    import torch
    heads, dim, page, n = 8, 256, 256, 300
    pages = (9 << 29) // (heads * dim * page)
    k = torch.zeros((pages * heads * page * dim,), dtype=torch.int8, device="cuda:0")
    v = torch.zeros_like(k)
    ks, vs = (torch.zeros((pages * heads * page,), device="cuda:0") for _ in range(2))
    c = pk.KvCache(k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), pk.I8, pages, page, heads, dim)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda:0")
    slots = (table[0].repeat_interleave(page) * page + torch.arange(page, device="cuda:0").repeat(2))[:n].int()
    wide = heads * dim
    x, y = (torch.randn((n, wide), device="cuda:0") for _ in range(2))
    pk.call("pk_gpu_kv_write_dev", do.ref(c), pk.F32, x.data_ptr(), wide, y.data_ptr(), wide, slots.data_ptr(), n,
            do.stream())
    rk, rv = torch.empty_like(x), torch.empty_like(y)
    pk.call("pk_gpu_kv_read_dev", do.ref(c), pk.F32, slots.data_ptr(), n, rk.data_ptr(), wide, rv.data_ptr(), wide,
            do.stream())
    q = torch.randn((1, wide), device="cuda:0")
    out = torch.zeros_like(q)
    lens = torch.tensor([n], dtype=torch.int32, device="cuda:0")
    floats = pk.load().pk_gpu_paged_attention_ws_floats(do.ref(c), 1, heads, n, 0)
    ws = torch.empty((floats + 4,), device="cuda:0")
    pk.call("pk_gpu_paged_attention_dev", do.ref(c), pk.F32, q.data_ptr(), wide, heads, table.data_ptr(), 2,
            lens.data_ptr(), 1, n, 0.0625, 0, out.data_ptr(), wide, None, ws.data_ptr(), floats, do.stream())
    torch.cuda.synchronize()

    class Rows:          # what the cache's rows stand for, by token
        pass
    r = Rows()
    r.heads, r.page, r.pages, r.dim, r.kind = heads, 1, n, dim, "int8"
    back = {"k": do.values(rk).reshape(n, heads, dim), "v": do.values(rv).reshape(n, heads, dim)}
    r.rows = back.__getitem__
    qh = do.values(q).reshape(1, heads, dim)
    want, _, a, s, xx = do.attention(r, qh, np.arange(n)[None], [n], n, 0.0625, 0)
    err = np.abs(do.values(out).reshape(1, heads, dim) - want)
    # the rows read back are rounded once more than the kernel's codes * scale
    assert np.all(err <= do.attention_bound(want, a, s, xx, n, dim, "int8", "f32") +
                  2.0 ** -23 * (1 + 2 * xx[..., None]) * a)


def test_no_sequences():
    cache = do.Cache("int8", 2, 1, 16, 64)
    pk.call("pk_gpu_paged_attention_dev", do.ref(cache.struct()), pk.F32, None, 64, 1, None, 2, None, 0, 32, 1.0, 0,
            None, 64, None, None, 0, do.stream())
