"""GPU: the attention of several new tokens where rows are many, against the plain 64-bit
form: every pairing of queries and caches, head sizes, lengths at the tiles' borders,
every rule, ragged batches, and sequences split over several workgroups."""
import re

import numpy as np
import pytest

import decode_oracle as do
from pkgpu import pk
from prompt_call import prompt, sides
from test_gpu_prompt_attention import rules_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


PAIRINGS = [("f16", "f16"), ("bf16", "bf16"), ("bf16", "f32"), ("int8", "bf16"), ("int8", "f16"), ("int8", "f32"),
            ("e4m3", "bf16"), ("e4m3", "f16"), ("e4m3", "f32"), ("e2m1", "bf16"), ("e2m1", "f16"), ("e2m1", "f32")]


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("kind,rows", PAIRINGS)
def test_pairings(kind, rows, dim):
    """A ragged batch, one sequence of which has no new token and one no other tokens; group 3 puts a token's heads
    into several waves."""
    rng = np.random.default_rng(dim)
    c = prompt(rng, kind, rows, 12, 3, dim, 16, [70, 0, 33, 129], [70, 40, 150, 131], tail=5, pad=64)
    assert c.many()
    c.check()
    assert c.cache.guards_whole()


@pytest.mark.parametrize("kind,rows,dim", [("bf16", "bf16", 128), ("f16", "f16", 64), ("e2m1", "bf16", 256), ("int8", "f32", 128),
                                           ("bf16", "f32", 256), ("e4m3", "bf16", 64), ("bf16", "bf16", 256)])
@pytest.mark.parametrize("how", [dict(window=1), dict(window=65), dict(docs=50), dict(docs=33, prefix=7), dict(prefix=100),
                                 dict(prefix=90, window=40), dict(cap=3.0), dict(slopes=True), dict(cap=20.0, slopes=True,
                                                                                                    docs=64, window=30)])
def test_rules(kind, rows, dim, how):
    rng = np.random.default_rng(dim + len(how))
    heads = 32
    c = prompt(rng, kind, rows, 16, 2, dim, 16, [130, 61], [200, 61], **rules_of(how, heads))
    assert c.many()
    c.check()


@pytest.mark.parametrize("dim,kind", [(64, "bf16"), (128, "bf16"), (256, "bf16"), (64, "int8"), (128, "e2m1"), (256, "e4m3")])
def test_lengths_at_the_borders_of_tiles(dim, kind):
    """Lengths, first tokens and row counts one off multiples of 16 to 128, large pages and small ones."""
    rng = np.random.default_rng(dim)
    for page in (16, 128):
        new = [1, 31, 32, 33, 63, 64, 65, 127, 128, 129]
        lens = [n + (i * 37) % 70 for i, n in enumerate(new)]
        c = prompt(rng, kind, "bf16", 8, 1, dim, page, new, lens)
        assert c.many()
        c.check()
        c = prompt(rng, kind, "bf16", 8, 1, dim, page, new, [x + 64 for x in new], first=lambda b, p: p // 16 * 16 - 1)
        c.check()


@pytest.mark.parametrize("group,kv", [(1, 40), (5, 8), (17, 3), (40, 1), (130, 1)])
def test_groups(group, kv):
    """Heads that share a key-value head, fewer and more than a tile has rows."""
    rng = np.random.default_rng(group)
    new = [110, 9] if group < 130 else [40, 9]
    c = prompt(rng, "bf16", "bf16", kv, group, 64, 16, new, [new[0], 80], slopes=np.linspace(0.01, 0.5, kv * group, dtype=np.float32))
    assert c.many()
    c.check()


def splits(c):
    """Chunks that the call asks a workspace for."""
    import ctypes
    lib = pk.load()
    rc = lib.pk_gpu_prompt_attention_dev(
        do.ref(c.st), do.FLOATS[c.rows], c.q.data_ptr(), c.ld, c.heads, c.table.data_ptr(), c.table.shape[1], c.lens.data_ptr(),
        c.starts.data_ptr(), c.B, c.n, c.max_new, c.max_len, ctypes.byref(c.rules), c.out.data_ptr(), c.ld, None, None, 0,
        do.stream())
    assert rc == -1
    need = int(re.search(r"workspace of (\d+) floats", lib.pk_gpu_last_error().decode()).group(1))
    each = c.n * c.heads * (c.cache.dim + 2)
    assert need % each == 0
    return need // each


SPLIT = [
    # kind, rows, kv, group, dim, new, lens, rules, chunks
    ("bf16", "bf16", 2, 4, 128, [200], [2600], {}, 9), ("int8", "bf16", 4, 4, 64, [300, 20], [3000, 1800], {}, 10),
    ("e2m1", "f32", 2, 3, 64, [400], [8000], dict(window=4000), 12),
    ("bf16", "bf16", 1, 2, 256, [500, 100, 0], [3100, 2000, 5], {}, 10),
    ("f16", "f16", 3, 3, 128, [230], [1500], dict(docs=700, prefix=300), 5),
    ("bf16", "f32", 1, 8, 64, [260], [5000], dict(cap=4.0), 16),
]


@pytest.mark.parametrize("kind,rows,kv,group,dim,new,lens,how,want", SPLIT)
def test_split_sequences(kind, rows, kv, group, dim, new, lens, how, want):
    rng = np.random.default_rng(dim + sum(lens))
    c = prompt(rng, kind, rows, kv, group, dim, 16, new, lens, tail=4, **rules_of(how, kv * group))
    assert c.many() and splits(c) == want, splits(c)
    c.table_h[0, 7] = -1
    import torch
    c.table.copy_(torch.from_numpy(c.table_h))
    c.check()
    # larger values than a chunk's sums hold: some chunks row by row, some not
    if kind == "bf16":
        c.cache.part("v")[:5] = 3e38
        c.check(more=2.0 ** -18)


def test_a_cache_past_4_gib():
    """The last pages of 4.5 GiB of keys and of values: element offsets beyond 32 bits."""
    import ctypes

    import more_oracle as mo
    import torch
    heads, dim, page, n = 8, 256, 256, 300
    pages = (9 << 28) // (heads * dim * page)
    k = torch.zeros((pages * heads * page * dim,), dtype=torch.bfloat16, device="cuda:0")
    v = torch.zeros_like(k)
    c = pk.KvCache(k.data_ptr(), v.data_ptr(), None, None, pk.BF16, pages, page, heads, dim)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device="cuda:0")
    slots = (table[0].repeat_interleave(page) * page + torch.arange(page, device="cuda:0").repeat(2))[:n].int()
    wide = heads * dim
    x, y, q = (torch.randn((n, wide), device="cuda:0").to(torch.bfloat16) for _ in range(3))
    pk.call("pk_gpu_kv_write_dev", do.ref(c), pk.BF16, x.data_ptr(), wide, y.data_ptr(), wide, slots.data_ptr(), n, do.stream())
    out = torch.zeros_like(q)
    lens, starts = (torch.tensor(t, dtype=torch.int32, device="cuda:0") for t in ([n], [0, n]))
    r = pk.AttentionRules(0.0625, 0.0, None, 0, None, None)
    floats = pk.load().pk_gpu_prompt_attention_ws_floats(do.ref(c), 1, n, heads, n, n, 0)
    ws = torch.empty((floats + 4,), device="cuda:0")
    pk.call("pk_gpu_prompt_attention_dev", do.ref(c), pk.BF16, q.data_ptr(), wide, heads, table.data_ptr(), 2, lens.data_ptr(),
            starts.data_ptr(), 1, n, n, n, ctypes.byref(r), out.data_ptr(), wide, None, ws.data_ptr(), floats, do.stream())
    torch.cuda.synchronize()

    class Rows:          # what the cache's rows stand for, by token
        pass
    held = Rows()
    held.heads, held.page, held.pages, held.dim, held.kind = heads, 1, n, dim, "bf16"
    held.rows = {"k": do.values(x).reshape(n, heads, dim), "v": do.values(y).reshape(n, heads, dim)}.__getitem__
    want = mo.Ruled(held, do.values(q).reshape(n, heads, dim), np.arange(n)[None], [n], [0, n], n, n, 0.0625)
    err = np.abs(do.values(out).reshape(n, heads, dim) - want.out)
    assert np.all(err <= want.bound("bf16", "bf16", 2.0 ** -8))


@pytest.mark.parametrize("B,most,kv,group,max_new,shift", [(64, 25, 3, 3, 60, 3), (65, 25, 3, 3, 60, 0), (150, 40, 2, 4, 60, 3),
                                                          (300, 9, 2, 2, 250, 0), (4200, 3, 1, 1, 130, 2), (4099, 2, 1, 1, 400, 0)])
def test_many_sequences(B, most, kv, group, max_new, shift):
    """As many row tiles as a sequence has rows, found among up to 64 sequences and among more; a bound on them
    that is not close, sequences without new tokens, and rows before the first sequence's."""
    import torch
    rng = np.random.default_rng(B)
    new = rng.integers(0, most + 1, B)
    new[::7], new[B // 2] = 0, most
    lens = new + rng.integers(0, 20, B)
    c = prompt(rng, "bf16", "bf16", kv, group, 64, 16, new.tolist(), lens.tolist(), max_new=max_new, tail=shift + 2,
               max_len=max_new + 20)
    c.starts_h = (c.starts_h + shift).astype(np.int32)
    c.starts.copy_(torch.from_numpy(c.starts_h))
    assert c.many()
    c.check()


def test_single_tokens_of_many_heads():
    """No starts: row b is sequence b's, 17 query heads to a key-value head."""
    rng = np.random.default_rng(17)
    c = prompt(rng, "int8", "bf16", 1, 17, 64, 16, [1] * 520, rng.integers(1, 60, 520).tolist())
    c.starts = c.starts_h = None
    assert c.many()
    c.check()


TWO = [(kind, rows, dim) for kind, rows in PAIRINGS for dim in (64, 128) if (kind, dim) != ("e2m1", 64)]


@pytest.mark.parametrize("kind,rows,dim", TWO)
def test_two_sides(kind, rows, dim):
    """Two waves with the same rows: a ragged batch in which some waves' halves see nothing, and values that leave a
    side's range, an absent page, a NaN in one side's tokens."""
    import torch
    rng = np.random.default_rng(dim + len(kind))
    c = prompt(rng, kind, rows, 11, 3, dim, 16, [70, 0, 33, 129], [470, 40, 450, 431], tail=5, pad=64)
    assert c.many() and sides(c) == 2
    c.check()
    c.table_h[0, [3, 4, 9]] = -1
    c.table.copy_(torch.from_numpy(c.table_h))
    c.check()
    if kind == "bf16":
        c.cache.part("v")[c.table_h[2, 6]] = 3e38
        c.check(more=2.0 ** -18)
        c.cache.part("v")[c.table_h[2, 6]] = 0.5
    assert c.cache.guards_whole()


@pytest.mark.parametrize("kind,rows,dim", [("bf16", "bf16", 128), ("f16", "f16", 64), ("e2m1", "f16", 128), ("int8", "f32", 128),
                                           ("bf16", "f32", 64), ("e4m3", "bf16", 64)])
@pytest.mark.parametrize("how", [dict(window=1, limit=600), dict(window=420), dict(docs=50), dict(docs=33, prefix=7),
                                 dict(prefix=100), dict(cap=3.0), dict(cap=20.0, slopes=True, docs=64, window=400)])
def test_rules_of_two_sides(kind, rows, dim, how):
    how = dict(how)
    how.pop("limit", None)
    rng = np.random.default_rng(dim + len(how))
    c = prompt(rng, kind, rows, 16, 2, dim, 16, [130, 61], [460, 61], **rules_of(how, 32))
    assert c.many() and (sides(c) == 2 or how.get("window") == 1)
    c.check()


@pytest.mark.parametrize("kind,rows,dim,chunks", [("bf16", "bf16", 64, 3), ("int8", "f16", 64, 3), ("bf16", "f32", 128, 3)])
def test_two_sides_and_chunks(kind, rows, dim, chunks):
    """Two chunks of 576 tokens, and one for rows that begin inside their first tile."""
    rng = np.random.default_rng(dim)
    kv = 32 if dim == 64 else 12
    c = prompt(rng, kind, rows, kv, 2, dim, 16, [400], [1100], tail=3)
    assert c.many() and sides(c) == 2
    assert splits(c) == chunks, splits(c)
    c.check()
    if kind == "bf16":
        c.cache.part("v")[5:9] = 3e38
        c.check(more=2.0 ** -18)


@pytest.mark.parametrize("new,kv", [(3, 2), (150, 16), (500, 16)])
def test_no_tokens_at_all(new, kv):
    """max_len 0 takes no page table; rows see nothing: zeros, lse -inf, and rows of no sequence stay."""
    import ctypes
    import torch
    cache = do.Cache("bf16", 2, kv, 16, 64)
    st = cache.struct()
    n = 2 * new + 1
    q = torch.randn((n, kv * 64), device="cuda:0").bfloat16()
    out, lse = torch.full_like(q, 3.0), torch.full((n, kv), 3.0, device="cuda:0")
    ints = lambda *a: torch.tensor(a, dtype=torch.int32, device="cuda:0")
    lens, starts = ints(5, 0), ints(0, new, 2 * new)
    r = pk.AttentionRules(1.0, 0.0, None, 0, None, None)
    pk.call("pk_gpu_prompt_attention_dev", do.ref(st), pk.BF16, q.data_ptr(), kv * 64, kv, None, 0, lens.data_ptr(),
            starts.data_ptr(), 2, n, new, 0, ctypes.byref(r), out.data_ptr(), kv * 64, lse.data_ptr(), None, 0, do.stream())
    torch.cuda.synchronize()
    assert bool((out[:-1] == 0).all()) and bool((out[-1] == 3).all())
    assert bool(torch.isneginf(lse[:-1]).all()) and bool((lse[-1] == 3).all())


@pytest.mark.parametrize("new,kv,kind,rows", [(5, 2, "int8", "bf16"), (130, 16, "bf16", "bf16"), (130, 16, "int8", "f32")])
def test_the_largest_and_smallest_of_a_rule(new, kv, kind, rows):
    """Ranges that begin behind everything or before it, and end so: as the documented maximum and minimum say."""
    rng = np.random.default_rng(new)
    big = 2 ** 31 - 1
    pick = lambda *v: (lambda b, p: np.where(b >= 0, np.array(v)[np.arange(len(p)) % len(v)], 0))
    c = prompt(rng, kind, rows, kv, 2, 64, 16, [new, new], [new + 300, new], first=pick(0, -big - 1, 7, big, 100, -1),
               until=pick(big, 0, -big - 1, big, 5))
    assert c.many() == (new > 5)
    c.check()
    c = prompt(rng, kind, rows, kv, 2, 64, 16, [new, new], [new + 300, new], window=new + 299, until=pick(big, 0, 90))
    c.check()
