"""Plain 64-bit (numpy) forms of the 4-bit cache, and the cache itself on the
device, beside decode_oracle's.  Nothing here calls the library's kernels."""
import numpy as np

import decode_oracle as do
from pkgpu import pk

GROUP = 32
LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])
KINDS = dict(do.KINDS, e2m1=pk.E2M1)


def codes4(x):
    """The documented rule: codes 0..15 of the last axis and a byte for each 32 of it."""
    x = np.asarray(x, np.float32)
    g = x.reshape(x.shape[:-1] + (-1, GROUP)).astype(np.float64)
    bad = ~np.isfinite(g).all(-1)
    a = np.where(bad, 0.0, np.abs(np.where(np.isfinite(g), g, 0)).max(-1))
    none = (a < do.TINY) | bad
    e = np.floor(np.log2(np.where(none, 1.0, a))) - 2          # a / 2^e in [4, 8)
    e = np.minimum(np.where(a > 7 * 2.0 ** e, e + 1, e), 125)
    y = np.abs(np.where(none[..., None], 0.0, np.where(np.isfinite(g), g, 0) / 2.0 ** e[..., None]))
    border = (LEVELS[1:] + LEVELS[:-1]) / 2                    # ties go to the even code
    up = np.where(np.arange(7) % 2 == 1, y[..., None] >= border, y[..., None] > border)
    code = up.sum(-1) + 8 * (np.signbit(g) & ~none[..., None])
    byte = np.where(bad, 255, np.where(none, 0, e + 127)).astype(np.uint8)
    return code.reshape(x.shape).astype(np.uint8), byte


def stand_for(code, byte):
    """float64 values of codes and bytes."""
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    unit = np.where(byte == 255, np.nan, 2.0 ** (byte.astype(np.float64) - 127))
    return v * np.repeat(unit, GROUP, -1)


class Cache4(do.Cache):
    """A 4-bit cache on the device, with guards."""

    def __init__(self, pages, heads, page, dim, seed=0, filled=True, spread=3):
        import torch
        self.kind, self.pages, self.heads, self.page, self.dim = "e2m1", pages, heads, page, dim
        rng = np.random.default_rng(seed)
        self.arrays = {}
        for name in ("k", "v"):
            x = rng.integers(0, 256, (pages, heads, page, dim // 2)) if filled else np.zeros((pages, heads, page, dim // 2))
            u = (rng.integers(127 - spread, 127, (pages, heads, page, dim // GROUP)) if filled
                 else np.zeros((pages, heads, page, dim // GROUP)))
            self._put(name, torch.from_numpy(x.astype(np.uint8)))
            self._put(name + "_scale", torch.from_numpy(u.astype(np.uint8)))

    def struct(self):
        p = {n: self.part(n).data_ptr() for n in self.arrays}
        return pk.KvCache(p["k"], p["v"], p["k_scale"], p["v_scale"], pk.E2M1, self.pages, self.page, self.heads, self.dim)

    def codes(self, name):
        """[slots][heads][dim] codes and [slots][heads][dim / 32] bytes."""
        b = self.part(name).cpu().numpy()
        c = np.stack([b & 15, b >> 4], -1).reshape(b.shape[:3] + (self.dim,))
        u = self.part(name + "_scale").cpu().numpy()
        return (c.transpose(0, 2, 1, 3).reshape(-1, self.heads, self.dim),
                u.transpose(0, 2, 1, 3).reshape(-1, self.heads, self.dim // GROUP))

    def rows(self, name):
        return stand_for(*self.codes(name))


def cache_of(kind, pages, heads, page, dim, seed=0, filled=True):
    if kind == "e2m1":
        return Cache4(pages, heads, page, dim, seed, filled)
    return do.Cache(kind, pages, heads, page, dim, seed, filled)


# ---- rotary positions ---------------------------------------------------------

def turned(x, pos, freqs, scale, rot, interleaved):
    """x [n][heads][dim] turned, in 64 bits, and per element what its tolerance is made of: |a| + |b| of its
    pair, times the scale (0 where it stays)."""
    x = np.asarray(x, np.float64)
    t = np.asarray(pos, np.float64)[:, None, None] * np.asarray(freqs, np.float64)
    c, s = np.cos(t) * np.float32(scale), np.sin(t) * np.float32(scale)
    i = np.arange(rot // 2)
    ia, ib = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
    a, b = x[..., ia], x[..., ib]
    y, size = x.copy(), np.zeros(x.shape)
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    size[..., ia] = size[..., ib] = (np.abs(a) + np.abs(b)) * abs(np.float64(np.float32(scale)))
    return y, size


def turned_bound(want, size, rows, far=1.0):
    """What the roundings add up to at most: cos and sin within 3 units in the last place of 1 or below (2^-24 each:
    the function's 2 and the first-order step's), the scale's product, an element's product and the sum: 6 of
    2^-24 of |a| + |b| times the scale; an angle of up to `far` radians is off by 2^-53 of it; the output's rounding."""
    return size * (6 * 2.0 ** -24 + far * 2.0 ** -53) + do.HALF[rows] * np.abs(want) * 1.01 + 2.0 ** -24 * (rows == "f16")


# ---- attention with rules -------------------------------------------------------

def ranges(lens, starts, rows, max_new, max_len, window=0, first=None, until=None):
    """Per row: sequence (-1: none), position, and the tokens [lo, hi) that it sees."""
    b_of, p_of, lo, hi = (np.full(rows, -1), np.zeros(rows, int), np.zeros(rows, int), np.zeros(rows, int))
    for b in range(len(lens)):
        s = min(max(int(starts[b]), 0), rows)
        n = min(min(max(int(starts[b + 1]), s), rows) - s, max_new)
        length = min(max(int(lens[b]), 0), max_len)
        for i in range(n):
            r, p = s + i, length - n + i
            b_of[r], p_of[r] = b, p
            lo[r] = max(0, int(first[r]) if first is not None else 0, p - window + 1 if window else 0)
            hi[r] = max(0, min(length, max(p + 1, int(until[r]) if until is not None else 0)))
    return b_of, p_of, lo, hi


class Ruled:
    """Outputs of the plain 64-bit form, and what their tolerances are made of."""

    def __init__(self, cache, q, table, lens, starts, max_new, max_len, scale, cap=0.0, slopes=None, window=0, first=None,
                 until=None, exact_tanh=False):
        rows, heads, dim = q.shape
        k, v = cache.rows("k"), cache.rows("v")
        group = heads // cache.heads
        self.live, pos, lo, hi = ranges(lens, starts, rows, max_new, max_len, window, first, until)
        self.out, self.a = np.zeros(q.shape), np.zeros(q.shape)
        self.lse, self.d = np.full((rows, heads), -np.inf), np.zeros((rows, heads))
        self.seen = np.zeros(rows, int)
        for b in sorted(set(self.live) - {-1}):
            mine = np.flatnonzero(self.live == b)
            n = hi[mine].max(initial=0)
            t = np.arange(n)
            page = table[b][t // cache.page] if n else t
            t = t[(page >= 0) & (page < cache.pages)]
            at = table[b][t // cache.page].astype(np.int64) * cache.page + t % cache.page if n else t
            p = pos[mine][:, None]
            see = (t >= lo[mine][:, None]) & (t < hi[mine][:, None])
            self.seen[mine] = see.sum(1)
            use = mine[see.any(1)]
            see, p = see[see.any(1)], p[see.any(1)]
            if not len(use):
                continue
            for h in range(heads):
                kk, vv = k[at, h // group], v[at, h // group]
                with np.errstate(all="ignore"):
                    s = scale * (q[use, h] @ kk.T)
                    x = abs(scale) * (np.abs(q[use, h]) @ np.abs(kk).T)
                    err = (dim + 8) * 2.0 ** -23 * x + 6 * 2.0 ** -24 * np.abs(s)
                    if cap:
                        s = cap * np.tanh(s / cap)
                        # tanh: 8 units of 1, or with exact_tanh 18 of its value (tanh_of)
                        err = err + 2.0 ** -24 * (18 * np.abs(s) if exact_tanh else 8 * cap) + 6 * 2.0 ** -24 * np.abs(s)
                    if slopes is not None:
                        bias = np.float64(slopes[h]) * np.abs(p - t)
                        s = s - bias
                        err = err + 4 * 2.0 ** -24 * (bias + np.abs(s))
                    s = np.where(see, s, -np.inf)
                    m = s.max(1, keepdims=True)
                    w = np.exp(s - m)
                    w = np.where(see, w, 0)
                    l = w.sum(1, keepdims=True)
                    # tokens that weigh less than 2^-40 of the heaviest move nothing, whatever their error
                    self.d[use, h] = np.where(w > 2.0 ** -40, err, 0).max(1)
                    vf = np.where(see.any(0)[:, None], vv, 0)
                    self.out[use, h], self.lse[use, h] = (w @ vf) / l, (m + np.log(l))[:, 0]
                    self.a[use, h] = (w @ np.abs(vf)) / l

    def bound(self, kind, rows, half_p):
        """As decode_oracle.attention_bound: scores' errors twice, exp2, a weight's rounding, sums, the output's."""
        n = np.maximum(self.seen, 1)[:, None]
        rel = 2 * self.d + 4 * 2.0 ** -23 + half_p + (n / 16 + 64 + n / 4 + 64) * 2.0 ** -23
        small = n[..., None] * 2.0 ** -32 * 8.0 if kind == "f16" else 0.0
        return (rel[..., None] * self.a * 1.01 + small + do.HALF[rows] * np.abs(self.out) * 1.01
                + 2.0 ** -24 * (rows == "f16"))

    def lse_bound(self):
        n = np.maximum(self.seen, 1)[:, None]
        return self.d + (n / 16 + 72) * 2.0 ** -23 + 4 * 2.0 ** -24 * np.where(np.isfinite(self.lse), np.abs(self.lse), 0)


def half_of_weights(kind, rows, many=False):
    """Half a step of what a softmax weight keeps in the second product: 16 bits, 24 for f32 outputs, over f16
    caches 22.  Where rows are many, 16-bit outputs over caches of their own type and bf16 ones over codes take
    one term: 8 bits in bf16 (half a step 2^-8 of the weight), 11 in f16 (2^-11)."""
    if many and rows == "bf16":
        return 2.0 ** -8
    if many and kind == "f16":
        return 2.0 ** -11
    return 2.0 ** -22 if kind == "f16" else {"bf16": 2.0 ** -16, "f16": 2.0 ** -16, "f32": 2.0 ** -24}[rows]
