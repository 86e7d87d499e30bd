"""One call of the attention with rules: its inputs on the device, its checks."""
import ctypes

import numpy as np

import decode_oracle as do
import more_oracle as mo
from pkgpu import pk


class Prompt:
    def __init__(self, cache, q, rows, table, lens, starts, max_new, max_len, scale, cap=0.0, slopes=None, window=0,
                 first=None, until=None, pad=0, lse=True):
        import torch
        self.cache, self.rows, self.max_new, self.max_len = cache, rows, max_new, max_len
        self.n, self.heads, dim = q.shape
        self.B, self.wide = len(lens), self.heads * dim
        self.ld = self.wide + pad
        self.q_h, self.table_h, self.lens_h, self.starts_h = q, np.asarray(table, np.int32), list(lens), starts
        self.how = dict(scale=scale, cap=cap, slopes=slopes, window=window, first=first, until=until)
        tt = do.torch_type(rows)
        self.q = torch.zeros((max(1, self.n), self.ld), dtype=tt, device="cuda:0")
        self.q[:self.n, :self.wide] = torch.from_numpy(q.reshape(self.n, -1)).to(tt).to("cuda:0")
        self.out = torch.full((self.n + 2, self.ld), 5.0, dtype=tt, device="cuda:0")
        self.lse = torch.full((self.n + 2, self.heads), 5.0, device="cuda:0") if lse else None
        put = lambda a, t=np.int32: None if a is None else torch.from_numpy(np.ascontiguousarray(a, t)).to("cuda:0")
        self.table, self.lens, self.starts = put(table), put(lens), put(starts)
        self.d = {"slopes": put(slopes, np.float32), "first": put(first), "until": put(until)}
        at = lambda n: self.d[n].data_ptr() if self.d[n] is not None else None
        self.rules = pk.AttentionRules(scale, cap, at("slopes"), window, at("first"), at("until"))
        self.st = cache.struct()
        self.floats = pk.load().pk_gpu_prompt_attention_ws_floats(do.ref(self.st), self.B, self.n, self.heads, max_new,
                                                                  max_len, window)
        self.ws = torch.full((self.floats + 64,), float("nan"), device="cuda:0")

    def enqueue(self, stream):
        pk.call("pk_gpu_prompt_attention_dev", do.ref(self.st), do.FLOATS[self.rows], self.q.data_ptr(), self.ld, self.heads,
                self.table.data_ptr(), self.table.shape[1], self.lens.data_ptr(),
                self.starts.data_ptr() if self.starts is not None else None, self.B, self.n, self.max_new, self.max_len,
                ctypes.byref(self.rules), self.out.data_ptr(), self.ld,
                self.lse.data_ptr() if self.lse is not None else None, self.ws.data_ptr(), self.floats, stream)

    def plain(self):
        starts = self.starts_h if self.starts_h is not None else np.arange(self.B + 1)
        return mo.Ruled(self.cache, self.q_h, self.table_h, self.lens_h, starts, self.max_new, self.max_len,
                        exact_tanh=self.rows == "f32", **self.how)

    def run(self, want):
        """The call's outputs; rows of no sequence, pitches and what lies behind are as they were."""
        import torch
        self.enqueue(do.stream())
        torch.cuda.synchronize()
        none = torch.from_numpy(want.live < 0).to("cuda:0")
        assert bool((self.out[self.n:] == 5).all()) and bool((self.out[:, self.wide:] == 5).all())
        assert bool((self.out[:self.n][none] == 5).all()) and bool(self.ws[self.floats:].isnan().all())
        if self.lse is not None:
            assert bool((self.lse[self.n:] == 5).all()) and bool((self.lse[:self.n][none] == 5).all())
        return do.values(self.out)[:self.n, :self.wide].reshape(self.n, self.heads, -1)

    def check(self, half_p=None, more=0.0):
        """`more`: relative to a, on top of the bound."""
        want = self.plain()
        got = self.run(want)
        live = want.live >= 0
        half_p = self.half_p() if half_p is None else half_p
        tol = want.bound(self.cache.kind, self.rows, half_p) + more * want.a
        err = np.abs(got - want.out)[live]
        assert np.all(err <= tol[live]), (float(np.nanmax(err / tol[live])), np.argwhere(~(err <= tol[live]))[:4].tolist())
        if self.lse is not None:
            lse = do.values(self.lse)[:self.n][live]
            none = np.isneginf(want.lse[live])
            assert np.array_equal(np.isneginf(lse), none)
            off = np.abs(lse[~none] - want.lse[live][~none])
            assert np.all(off <= want.lse_bound()[live][~none] + more)
        return got

    def half_p(self):
        return mo.half_of_weights(self.cache.kind, self.rows, self.many())

    def many(self):
        """Whether the call takes the kernel of many rows."""
        new = min(self.max_new, self.n) if self.starts is not None else 1
        return many_rows(self.cache.kind, self.rows, self.cache.heads, self.heads // self.cache.heads, self.B, new, self.max_len,
                         self.how["window"])


def sides(c):
    """Whether two waves share rows in the kernel of many rows: its rule for what a call's tiles are."""
    kind, rows, dim, heads = c.cache.kind, c.rows, c.cache.dim, c.cache.heads
    if dim == 256 or (dim == 64 and kind == "e2m1"):
        return 1
    if dim == 128 and rows == "f32" and kind != "e2m1":
        return 2
    group, new = c.heads // heads, min(c.max_new, c.n)
    window = c.how["window"] if c.how["window"] < c.max_len else 0
    span = min(window + new + 30, c.max_len) if window else c.max_len
    pairs = min(-(-new * group // 128) * c.B, c.n * group // 128 + c.B) * heads
    split = -(-c.n * group // 128) * heads
    most = (1024 if c.how["first"] is not None and rows != "f32" else 512) if dim == 64 else 512 if span >= 1024 else 256
    slots = 768 if dim == 64 and rows != "f32" else 512
    cuts = 1 if split >= 256 else max(1, min(slots // split, span // (256 if split <= 64 else 512), 64))
    return 2 if pairs <= most and span >= 384 and (pairs >= 192 or cuts == 1) else 1


def many_rows(kind, rows, kv, group, B, new, max_len, window):
    """The rule: by the rows of a sequence and key-value head, the 16-row tiles of all and the tokens that a
    tile may see."""
    each = new * group
    tiles = -(-each // 16) * B * kv
    window = window if window < max_len else 0
    span = min(window + new + 30, max_len) if window else max_len
    narrow = rows != "f32" and kind in ("f16", "bf16")
    wide = rows == "f32" or kind == "e2m1"
    few = (each <= 16 or (each <= 32 and (B * kv < 256 or span >= (512 if wide else 1536))) or
           (32 < each <= 48 and wide and B * kv < 512) or
           (tiles <= (256 if narrow else 512) and
            tiles * span <= (160 << 10 if narrow else 1 << 20 if kind == "e2m1" and rows != "f32" else 512 << 10)))
    return not few


def prompt(rng, kind, rows, kv, group, dim, page, new, lens, max_new=None, max_len=None, tail=0, pad=0, scale=None, seed=1,
           spare=1, **how):
    """A call with new[b] rows for each sequence, `tail` rows of padding behind, distinct pages in any order."""
    B = len(lens)
    max_len = max_len or max(1, max(lens))
    max_new = max_new or max(1, max(new))
    per = (max_len + page - 1) // page
    cache = mo.cache_of(kind, B * per + spare, kv, page, dim, seed=seed)
    table = rng.permutation(cache.pages)[:B * per].reshape(B, per).astype(np.int32)
    for b, n in enumerate(lens):
        table[b, (max(0, n) + page - 1) // page:] = 1 << 30           # entries nothing may read
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    n = int(starts[-1]) + tail
    q = do.rounded(rng.normal(0, 1, (n, kv * group, dim)), rows).astype(np.float64)
    for name in ("first", "until"):
        if callable(how.get(name)):
            live, pos, _, _ = mo.ranges(lens, starts, n, max_new, max_len)
            how[name] = np.where(live >= 0, how[name](live, pos), 0).astype(np.int32)
    return Prompt(cache, q, rows, table, lens, starts, max_new, max_len, scale or dim ** -0.5, pad=pad, **how)
