"""GPU: attention of several new tokens per sequence with caps, biases, windows,
documents and prefixes, against the plain 64-bit form within the bound that its
roundings add up to (more_oracle.Ruled)."""
import numpy as np
import pytest

import decode_oracle as do
import more_oracle as mo
from pkgpu import pk
from prompt_call import Prompt, prompt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


def slopes(heads):
    return np.exp2(-8.0 * np.arange(1, heads + 1) / heads).astype(np.float32)


FEW = [0, 1, 2, 3, 5]
CASES = [
    # kind, rows, kv, group, dim, page, new, lens, rules
    # single tokens
    ("int8", "bf16", 2, 4, 128, 16, [1] * 6, [1, 2, 31, 32, 33, 300], dict(cap=30.0)),
    ("bf16", "f32", 1, 3, 64, 32, [1] * 4, [700, 1, 64, 65], dict(slopes=True, window=100)),
    ("e2m1", "f16", 2, 8, 128, 16, [1, 0, 1], [4000, 5, 77], dict(cap=5.0, slopes=True)),
    # a few each
    ("bf16", "bf16", 2, 4, 128, 16, FEW, [4, 1, 500, 33, 64], {}),
    ("f16", "f16", 1, 5, 64, 64, FEW, [0, 7, 129, 3, 1000], dict(window=3)),
    ("e4m3", "f32", 3, 1, 256, 16, FEW, [9, 10, 11, 12, 400], dict(cap=10.0)),
    ("int8", "f16", 1, 20, 128, 32, [3, 2], [900, 40], dict(slopes=True)),
    ("e2m1", "f32", 2, 2, 64, 16, [7, 4], [5000, 3000], dict(window=2500)),
    # prompts
    ("bf16", "bf16", 2, 2, 128, 16, [130], [130], {}),
    ("bf16", "f32", 1, 2, 128, 16, [257, 64, 1], [300, 64, 129], dict(cap=20.0)),
    ("f16", "f16", 2, 4, 64, 32, [100, 0, 33], [100, 0, 700], dict(window=50)),
    ("int8", "bf16", 1, 3, 128, 64, [200, 65], [513, 65], dict(slopes=True, cap=50.0)),
    ("e4m3", "f16", 2, 1, 64, 16, [150], [150], dict(docs=40)),
    ("e2m1", "bf16", 1, 4, 256, 16, [90, 31], [200, 31], dict(docs=20, prefix=5)),
    ("bf16", "bf16", 1, 1, 256, 16, [70, 70], [90, 70], dict(prefix=33, window=60)),
    ("int8", "f32", 1, 2, 64, 16, [300], [1000], dict(docs=100, prefix=30, cap=8.0, slopes=True)),
    ("bf16", "f32", 1, 1, 256, 32, [100], [128], {}),
    ("e4m3", "bf16", 1, 2, 128, 16, [129, 128, 127], [129, 1000, 127], dict(window=1)),
    ("f16", "f16", 1, 7, 256, 16, [40], [300], dict(prefix=400)),
    ("e2m1", "f16", 1, 1, 128, 128, [260], [260], {}),
    ("int8", "bf16", 8, 1, 64, 16, [65], [65], {}),
]


def rules_of(how, heads):
    how = dict(how)
    docs, prefix = how.pop("docs", 0), how.pop("prefix", 0)
    if how.get("slopes"):
        how["slopes"] = slopes(heads)
    if docs:
        how["first"] = lambda b, p: p // docs * docs
    if prefix:
        how["until"] = (lambda b, p: np.minimum(p // docs * docs + prefix, p // docs * docs + docs)) if docs else \
            (lambda b, p: np.full_like(p, prefix))
    return how


@pytest.mark.parametrize("kind,rows,kv,group,dim,page,new,lens,how", CASES)
def test_against_plain_form(kind, rows, kv, group, dim, page, new, lens, how):
    rng = np.random.default_rng(dim + sum(lens))
    c = prompt(rng, kind, rows, kv, group, dim, page, new, lens, tail=3, pad=64, **rules_of(how, kv * group))
    c.check()
    assert c.cache.guards_whole()


@pytest.mark.parametrize("rows,kind", [("bf16", "bf16"), ("f32", "int8"), ("f16", "f16"), ("bf16", "e2m1")])
@pytest.mark.parametrize("new,length,kv", [(1, 50, 2), (4, 50, 2), (90, 140, 2), (90, 140, 16)])
def test_rows_that_see_nothing(rows, kind, new, length, kv):
    """Empty ranges in the middle, first past the query, absent pages: zeros, and lse -inf."""
    rng = np.random.default_rng(new)
    first = lambda b, p: np.where(p % 3 == 0, 1 << 30, np.where(p % 3 == 1, -7, p))
    c = prompt(rng, kind, rows, kv, 2, 128, 16, [new, new, 0, new], [length, length, 9, length], first=first)
    assert c.many() == (kv == 16)
    c.table_h[1] = -1                                     # nothing of sequence 1
    c.table_h[3, 1:3] = c.cache.pages + 5
    c.table.copy_(do_int(c.table_h))
    got = c.check()
    want = c.plain()
    none = (want.seen == 0) & (want.live >= 0)
    assert none.any() and np.all(got[none] == 0)


def do_int(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, np.int32))


def test_one_row_each_without_starts():
    rng = np.random.default_rng(3)
    B, kv, group, dim, page = 5, 2, 3, 64, 16
    lens = [40, 0, 1, 99, 64]
    cache = mo.cache_of("int8", B * 7, kv, page, dim)
    table = np.arange(B * 7).reshape(B, 7)
    q = do.rounded(rng.normal(0, 1, (B, kv * group, dim)), "f32").astype(np.float64)
    for max_new in (1, 9):
        Prompt(cache, q, "f32", table, lens, None, max_new, 100, 0.125, cap=4.0).check()


def test_starts_lengths_and_counts_out_of_range():
    """What lies outside of the rows, of max_new and of max_len is not there."""
    rng = np.random.default_rng(4)
    B, kv, dim, page, rows = 6, 1, 64, 16, 40
    cache = mo.cache_of("bf16", B * 5, kv, page, dim)
    table = np.arange(B * 5).reshape(B, 5)
    q = do.rounded(rng.normal(0, 1, (rows, 2, dim)), "bf16").astype(np.float64)
    starts = np.array([-5, 3, 3, 20, 1 << 30, 1 << 30, -1], np.int32)       # the fourth's end is past the rows
    for max_new in (2, 9, 100):
        for lens in ([3, 10, 80, 17, 60, 60], [1 << 30, -4, 2, 75, 80, 0]):
            Prompt(cache, q, "bf16", table, lens, starts, max_new, 80, 0.125, lse=max_new > 2).check()


@pytest.mark.parametrize("kind,rows", [("int8", "bf16"), ("e4m3", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("e2m1", "bf16"),
                                       ("e2m1", "f16")])
@pytest.mark.parametrize("new,kv", [(3, 2), (150, 2), (150, 16)])
def test_masked_places_may_hold_anything(kind, rows, new, kv):
    """NaN and infinities wherever no row looks: behind the lengths, before the window, in absent pages' and other
    documents' places."""
    import torch
    rng = np.random.default_rng(new)
    lens = [250, 200]
    c = prompt(rng, kind, rows, kv, 2, 64, 16, [new, new], lens, window=40, first=lambda b, p: p // 32 * 32, spare=4)
    assert c.many() == (kv == 16)
    c.table_h[0, 10] = -1
    c.table.copy_(do_int(c.table_h))
    want = c.plain()
    live, pos, lo, hi = mo.ranges(lens, c.starts_h, c.n, c.max_new, c.max_len, 40, c.how["first"])
    seen = np.zeros((c.cache.pages, 16), bool)
    for r in range(c.n):
        for t in range(lo[r], hi[r]):
            id_ = c.table_h[live[r], t // 16]
            if 0 <= id_ < c.cache.pages:
                seen[id_, t % 16] = True
    assert not seen.all()
    fill(c.cache, ~seen)
    got = c.run(want)
    assert np.isfinite(got).all()
    tol = want.bound(kind, rows, c.half_p())
    assert np.all(np.abs(got - want.out) <= tol)
    if new == 3:
        assert torch.isfinite(c.lse[:c.n]).all()


def fill(cache, hide):
    """NaN and infinities (codes: -128, NaN scales and bytes) in the places of `hide` [pages][page]."""
    import torch
    hide = torch.from_numpy(hide).to("cuda:0")[:, None, :]
    for name in cache.arrays:
        p = cache.part(name)
        h = hide if p.dim() == 3 else hide[..., None]
        if p.dtype in (torch.int8, torch.uint8):
            p.copy_(torch.where(h, torch.full_like(p, -128 if p.dtype == torch.int8 else 255), p))
        elif p.dtype == torch.float8_e4m3fn:
            b = p.view(torch.uint8)
            b.copy_(torch.where(h, torch.full_like(b, 0x7F), b))
        else:
            alt = torch.where(torch.rand(p.shape, device="cuda:0") < 0.5, float("nan"), float("inf")).to(p.dtype)
            p.copy_(torch.where(h, alt, p))


@pytest.mark.parametrize("kind,rows", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("e2m1", "bf16"), ("e4m3", "bf16"),
                                       ("int8", "f16")])
@pytest.mark.parametrize("new,length,kv", [(4, 60, 2), (140, 140, 2), (140, 140, 32)])
def test_a_token_that_only_later_rows_see_may_hold_anything(kind, rows, new, length, kv):
    """A NaN or an infinity in a new token's value does not reach the rows before it; it does reach the later ones."""
    rng = np.random.default_rng(5)
    c = prompt(rng, kind, rows, kv, 2, 64, 16, [new], [length])
    assert c.many() == (kv == 32)
    at = length - new // 2                                    # the token
    want = c.plain()
    page, off = c.table_h[0, at // 16], at % 16
    v = c.cache.part("v")
    if kind in ("e2m1", "int8", "e4m3"):
        sc = c.cache.part("v_scale")
        sc[page, :, off] = 255 if kind == "e2m1" else float("nan")
    else:
        v[page, 0, off, 3], v[page, 1, off, 5] = float("nan"), -float("inf")
    got = c.run(want)
    before = np.arange(c.n) + length - new < at
    tol = want.bound(kind, rows, c.half_p())
    assert np.all(np.abs(got - want.out)[before] <= tol[before])
    if kind in ("e2m1", "int8", "e4m3"):
        assert np.isnan(got[~before]).all()
    else:
        assert np.isnan(got[~before][:, :2, 3]).all() and np.all(got[~before][:, 2:4, 5] == -np.inf)
        rest = np.abs(got - want.out) <= tol
        rest[:, :2, 3] = rest[:, 2:4, 5] = True
        assert rest.all()


LARGE = 3.3e38


@pytest.mark.parametrize("kind,rows,dim,kv,new,lens", [
    ("bf16", "bf16", 128, 1, [5], [700]), ("bf16", "f32", 64, 1, [3, 2], [5000, 31]), ("bf16", "bf16", 64, 1, [100], [300]),
    ("int8", "bf16", 128, 1, [70], [200]), ("e4m3", "f32", 64, 1, [66], [66]), ("bf16", "f32", 256, 1, [40], [90]),
    ("bf16", "bf16", 128, 16, [150], [150]), ("int8", "bf16", 64, 32, [140], [200]), ("bf16", "f32", 64, 32, [140], [150]),
])
def test_values_near_the_largest_float(kind, rows, dim, kv, new, lens):
    """Outputs are means of them, so they stay finite (weights 2^-18 off, as in the one-token attention)."""
    import torch
    rng = np.random.default_rng(dim)
    c = prompt(rng, kind, rows, kv, 2, dim, 16, new, lens)
    assert c.many() == (kv > 1)
    v = c.cache.part("v")
    size = rng.uniform(0.2, 1.0, tuple(v.shape)) * rng.choice([-1.0, 1.0], tuple(v.shape))
    top = do.TOP.get(kind, LARGE)
    x = torch.from_numpy((size * top).astype(np.float32)).to("cuda:0")
    x = (x.round() if kind == "int8" else x).to(v.dtype)
    v.view(torch.uint8).copy_(x.view(torch.uint8))
    if kind in do.TOP:
        c.cache.part("v_scale").fill_(LARGE / top)
    c.check(more=2.0 ** -18)


def test_large_flat_and_negative_scores():
    rng = np.random.default_rng(8)
    for scale in (20.0, -3.0, 0.0):
        for new, kv, rows in ((3, 1, "f32"), (200, 1, "f32"), (200, 16, "bf16"), (200, 32, "f32")):
            c = prompt(rng, "bf16", rows, kv, 2, 64, 16, [new], [300], scale=scale or None)
            assert c.many() == (kv > 1)
            c.rules.scale = c.how["scale"] = scale
            c.check()


def test_caps_small_and_large():
    rng = np.random.default_rng(9)
    for cap in (1e-3, 0.5, 1e4):
        for rows, new, kv in (("f32", 2, 1), ("f32", 90, 1), ("bf16", 90, 1), ("bf16", 90, 32), ("f32", 90, 64)):
            c = prompt(rng, "bf16", rows, kv, 2, 64, 16, [new], [200], cap=cap, scale=1.0)
            assert c.many() == (kv > 1)
            c.check()


def test_no_rows_is_no_work():
    import ctypes
    cache = do.Cache("int8", 2, 1, 16, 64)
    r = pk.AttentionRules(1.0, 0.0, None, 0, None, None)
    for B, rows, new in ((0, 4, 4), (3, 0, 4), (3, 4, 0)):
        pk.call("pk_gpu_prompt_attention_dev", do.ref(cache.struct()), pk.F32, None, 64, 1, None, 2, None, None, B, rows, new,
                32, ctypes.byref(r), None, 64, None, None, 0, do.stream())


def test_two_graphs_and_a_second_stream():
    """Captured calls with workspaces of their own, replayed side by side with changing lengths and starts, give
    what eager calls give, bit for bit."""
    import torch
    rng = np.random.default_rng(12)
    calls, graphs, streams = [], [], []
    for i, (new, kind, kv) in enumerate(((4, "int8", 2), (70, "bf16", 2), (70, "bf16", 16), (1, "e2m1", 2), (1100, "int8", 2))):
        c = prompt(rng, kind, "bf16", kv, 2, 64, 16, [new, new], [1500, 1200], max_new=new, tail=2, cap=9.0, seed=20 + i)
        assert c.many() == (kv == 16 or new == 1100)
        c.table_h[:] = rng.permutation(c.cache.pages)[:c.table_h.size].reshape(c.table_h.shape)
        c.table.copy_(do_int(c.table_h))
        calls.append(c)
        s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            c.enqueue(s.cuda_stream)
        graphs.append(g)
        streams.append(s)
    for lens, part in (([1500, 1200], 1.0), ([1500, 1499], 0.5), ([70, 700], 1.0)):
        want = []
        for c in calls:
            n = max(1, int(c.max_new * part))
            c.lens_h, c.starts_h = lens, np.array([0, n, 2 * n], np.int32)
            c.lens.copy_(do_int(lens))
            c.starts.copy_(do_int(c.starts_h))
            c.out.fill_(5.0)
            c.lse.fill_(5.0)
            want.append(c.check())
            c.out.fill_(5.0)
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for c, w in zip(calls, want):
            assert np.array_equal(do.values(c.out)[:c.n, :c.wide].reshape(w.shape), w)


def test_the_same_call_gives_the_same_bits():
    import torch
    rng = np.random.default_rng(3)
    for new, kind in ((3, "bf16"), (200, "int8"), (200, "bf16")):
        c = prompt(rng, kind, "bf16", 1, 4, 128, 16, [new, new], [5000, 2222], window=4000)
        assert c.floats > 0
        want = c.plain()
        first = c.run(want)
        for i in range(5):
            c.ws[:c.floats] = torch.randn((c.floats,), device="cuda:0") * 10.0 ** (i - 3)
            assert np.array_equal(c.run(want), first)


@pytest.mark.parametrize("B,kv,group,new,lens,kind,rows", [
    # more workgroups of whole sequences than CUs, one tile of rows each and two; 37 pairs beyond whole groups of 32
    (37, 5, 4, 8, 700, "bf16", "f32"), (41, 7, 3, 1, 1400, "int8", "bf16"), (90, 3, 16, 2, 690, "e2m1", "bf16"),
    (43, 6, 4, 7, 1600, "bf16", "bf16"), (300, 1, 20, 1, 600, "e2m1", "f32")])
def test_batches_longer_than_the_card(B, kv, group, new, lens, kind, rows):
    """Ragged batches: longest sequences first where they are long for their number, and the tiles of a key-value
    head in turn; some sequences without new tokens, some without any."""
    rng = np.random.default_rng(B)
    n = rng.integers(0, new + 1, B)
    n[0] = new
    ln = np.maximum(n, rng.integers(0, lens + 1, B))
    ln[1], n[2], ln[2] = lens, 0, 0
    c = prompt(rng, kind, rows, kv, group, 64, 16, n.tolist(), ln.tolist(), tail=1, max_len=lens, max_new=new)
    assert not c.many()
    c.check()
