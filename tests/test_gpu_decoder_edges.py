"""GPU: calls that the decoder operators' documentation allows at its ends: 4-bit groups of any byte, pages that
sequences share, bounds far above what a batch holds, several calls at once."""
import numpy as np
import pytest
import torch

import decode_oracle as do
import more_oracle as mo
from pkgpu import pk
from prompt_call import Prompt, prompt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


def test_groups_of_every_byte():
    """Each code with each unit from 2^-127 to 2^127; what passes the largest float is infinite, byte 255 NaN."""
    dim, page, pages = 64, 16, 8
    cache = mo.Cache4(pages, 1, page, dim, filled=False)
    codes = np.tile(np.arange(16, dtype=np.uint8), dim // 16)
    packed = torch.from_numpy((codes[::2] | codes[1::2] << 4).astype(np.uint8)).to("cuda:0")
    for name in ("k", "v"):
        cache.part(name)[:] = packed
        cache.part(name + "_scale")[:] = torch.arange(256, dtype=torch.uint8, device="cuda:0").view(pages, 1, page, 2)
    slots = torch.arange(128, dtype=torch.int32, device="cuda:0")
    out = [torch.zeros((128, dim), device="cuda:0") for _ in range(2)]
    pk.call("pk_gpu_kv_read_dev", do.ref(cache.struct()), pk.F32, slots.data_ptr(), 128, out[0].data_ptr(), dim, out[1].data_ptr(),
            dim, do.stream())
    torch.cuda.synchronize()
    with np.errstate(over="ignore"):
        want = mo.stand_for(np.tile(codes, (128, 1)), np.arange(256, dtype=np.uint8).reshape(128, 2)).astype(np.float32)
    for y in out:
        y = y.cpu().numpy()
        bad = ~((y == want) | (np.isnan(y) & np.isnan(want)))
        assert not bad.any(), (np.argwhere(bad)[:4], y[bad][:4], want[bad][:4])


@pytest.mark.parametrize("rows", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("new,kv", [(1, 2), (3, 2), (140, 32)])
def test_attention_over_groups_of_far_bytes(rows, new, kv):
    """Keys and values with units of 2^-90 to 2^15; values up to 2^124 in bf16 and f32."""
    rng = np.random.default_rng(new)
    c = prompt(rng, "e2m1", rows, kv, 2, 64, 16, [new], [150], scale=0.01)
    assert c.many() == (new > 3)
    top = 142 if rows == "f16" else 248
    for name, lo, hi in (("k_scale", 37, 131), ("v_scale", 60, top)):
        p = c.cache.part(name)
        p.copy_(torch.from_numpy(rng.integers(lo, hi, tuple(p.shape)).astype(np.uint8)))
    c.check(more=2.0 ** -18)


@pytest.mark.parametrize("kind,rows", [("bf16", "bf16"), ("int8", "f32"), ("e2m1", "f16")])
@pytest.mark.parametrize("new,kv", [(2, 2), (90, 32)])
def test_pages_that_sequences_share(kind, rows, new, kv):
    """A common prefix in the same pages, once in the middle of a page table of its own order, one page twice."""
    rng = np.random.default_rng(7)
    c = prompt(rng, kind, rows, kv, 2, 64, 16, [new] * 3, [400, 300, 200])
    assert c.many() == (new > 2)
    c.table_h[1, :6] = c.table_h[0, :6]
    c.table_h[2, 3:6] = c.table_h[0, 2:5]
    c.table_h[2, 8] = c.table_h[2, 7]
    c.table.copy_(torch.from_numpy(c.table_h))
    c.check()


@pytest.mark.parametrize("kind,rows", [("bf16", "bf16"), ("f16", "f16"), ("int8", "f32"), ("e2m1", "bf16")])
@pytest.mark.parametrize("new,kv,window", [(1, 2, 0), (3, 2, 70), (150, 2, 0), (150, 16, 0), (150, 16, 40), (150, 1, 2 ** 31 - 1)])
def test_bounds_far_above_the_batch(kind, rows, new, kv, window):
    """max_len 2^30 and max_new in the thousands, over some hundred tokens."""
    rng = np.random.default_rng(new)
    most = 1 << 30
    cache = mo.cache_of(kind, 40, kv, 16, 64, seed=2)
    lens, news = [new + 130, new, 0], [new, new // 2, 0]
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    q = do.rounded(rng.normal(0, 1, (int(starts[-1]) + 2, kv * 2, 64)), rows).astype(np.float64)
    table = np.full((3, 1024), 1 << 29, np.int32)
    table[:, :20] = rng.permutation(cache.pages)[:20]
    Prompt(cache, q, rows, table, lens, starts, 5000, 1 << 14, 0.125, window=window).check()       # 1024 pages of 16
    big = mo.cache_of(kind, 3, 1, 1024, 64, seed=3)
    wide = np.full((3, most >> 10), -1, np.int32)
    wide[:, 0] = [2, 0, 1]
    q = do.rounded(rng.normal(0, 1, (int(starts[-1]) + 2, 2, 64)), rows).astype(np.float64)
    Prompt(big, q, rows, wide, lens, starts, 5000, most, 0.125, window=window).check()


def test_calls_at_once():
    """Calls of both kernels, and writes to other pages, on streams of their own at the same time, again and again."""
    rng = np.random.default_rng(11)
    calls = [prompt(rng, kind, rows, kv, 4, dim, 16, new, lens, seed=i) for i, (kind, rows, kv, dim, new, lens) in enumerate((
        ("bf16", "bf16", 4, 128, [300, 200], [900, 300]), ("int8", "bf16", 2, 64, [3, 4], [4000, 3000]),
        ("e2m1", "f16", 4, 128, [1, 1], [5000, 70]), ("f16", "f16", 2, 256, [130], [2000]), ("int8", "f32", 8, 64, [700], [900])))]
    want = [c.check() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    for c in calls:
        c.out.fill_(5.0)
    torch.cuda.synchronize()
    for _ in range(20):
        for c, s in zip(calls, streams):
            c.enqueue(s.cuda_stream)
    torch.cuda.synchronize()
    for c, w in zip(calls, want):
        assert np.array_equal(do.values(c.out)[:c.n, :c.wide].reshape(w.shape), w)
