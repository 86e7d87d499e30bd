"""Plain 64-bit (numpy) forms of the decoder operators, and the small helpers
their tests share.  Nothing here calls the library's kernels."""
import ctypes

import numpy as np

from pkgpu import pk

FLOATS = {"f32": pk.F32, "f16": pk.F16, "bf16": pk.BF16}
KINDS = dict(FLOATS, int8=pk.I8, e4m3=pk.E4M3)
TOP = {"int8": 127.0, "e4m3": 448.0}
# half a step of a type, relative to the value: what one rounding is off by at most
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8, "e4m3": 2.0 ** -4}
TINY = 2.0 ** -100


def torch_type(name):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
            "int8": torch.int8, "e4m3": torch.float8_e4m3fn}[name]


def rounded(x, name):
    """float32 array rounded to a type and back (the CPU's conversions)."""
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch_type(name)).float().numpy()


def values(t):
    """A torch tensor of any of the types as float64 numpy."""
    return t.detach().cpu().float().double().numpy()


def codes(x, kind):
    """The documented fp32 formula: codes (as the values they are) and scales of the last axis's rows."""
    x = np.asarray(x, np.float32)
    top = np.float32(TOP[kind])
    a = np.abs(x).max(-1)
    bad = ~np.isfinite(x).all(-1)
    none = (a < np.float32(TINY)) | bad
    with np.errstate(all="ignore"):
        inv = np.where(none, np.float32(0), top / a).astype(np.float32)
        scale = np.where(none, np.float32(0), a / top).astype(np.float32)
        scale = np.minimum(scale, np.float32(float.fromhex("0x1.020406p+121")))   # 127 times it is finite
        y = np.where(none[..., None], np.float32(0), x * inv[..., None]).astype(np.float32)
    scale = np.where(bad, np.float32(np.nan), scale)
    return (np.rint(y) if kind == "int8" else rounded(y, "e4m3")), scale


def code_bound(x, kind):
    """How far code * scale may be from x (64 bits): half a step of the code, at
    the row's unit u = max|x| / top, plus the three fp32 roundings of inv, x * inv
    and scale, each at most 2^-24 of a value of at most max|x| (3.01: with their
    products)."""
    x = np.asarray(x, np.float64)
    if kind not in TOP:                     # a 16-bit cache: one rounding
        return HALF[kind] * np.abs(x)
    a = np.abs(x).max(-1, keepdims=True)
    u = a / TOP[kind]
    if kind == "int8":
        half = 0.5 * u * np.ones_like(x)
    else:  # 3 bits behind the leading one; the smallest exponent is -6
        m = np.maximum(np.abs(x) / np.where(u == 0, 1, u), 2.0 ** -6)
        # the quotient may round up over a power of two: its step then is the larger one
        half = 0.5 * u * 2.0 ** (np.floor(np.log2(m * (1 + 2.0 ** -22))) - 3)
    return half + 3.01 * 2.0 ** -24 * a


class Cache:
    """A cache on the device (torch tensors) with guard elements on both sides of each array."""

    GUARD = 64

    def __init__(self, kind, pages, heads, page, dim, seed=0, filled=True):
        import torch
        self.kind, self.pages, self.heads, self.page, self.dim = kind, pages, heads, page, dim
        rng = np.random.default_rng(seed)
        self.arrays = {}
        shape = (pages, heads, page, dim)
        for name in ("k", "v"):
            if not filled:
                x = np.zeros(shape, np.float32)
            elif kind == "int8":
                x = rng.integers(-127, 128, shape).astype(np.float32)
            elif kind == "e4m3":
                x = np.clip(rng.normal(0, 120, shape), -448, 448)
            else:
                x = rng.normal(0, 1, shape)
            self._put(name, torch.from_numpy(np.asarray(x, np.float32)).to(torch_type(kind)))
            if kind in TOP:
                sc = rng.uniform(0.5, 2.0, shape[:3]) / TOP[kind] if filled else np.zeros(shape[:3])
                self._put(name + "_scale", torch.from_numpy(np.asarray(sc, np.float32)))

    def _put(self, name, t):
        import torch
        flat = t.contiguous().view(torch.uint8).reshape(-1)
        guard = torch.full((self.GUARD,), 0x5A, dtype=torch.uint8)
        whole = torch.cat([guard, flat, guard]).to("cuda:0")
        self.arrays[name] = (whole, t.shape, t.dtype)

    def part(self, name):
        whole, shape, dtype = self.arrays[name]
        return whole[self.GUARD:-self.GUARD].view(dtype).view(shape)

    def guards_whole(self):
        return all(bool((w[:self.GUARD] == 0x5A).all() and (w[-self.GUARD:] == 0x5A).all())
                   for w, _, _ in self.arrays.values())

    def struct(self):
        p = {n: self.part(n).data_ptr() for n in self.arrays}
        return pk.KvCache(p["k"], p["v"], p.get("k_scale"), p.get("v_scale"), KINDS[self.kind],
                          self.pages, self.page, self.heads, self.dim)

    def rows(self, name):
        """float64 [slots][heads][dim], what the cache's rows stand for."""
        x = values(self.part(name)).transpose(0, 2, 1, 3).reshape(-1, self.heads, self.dim)
        if self.kind in TOP:
            sc = values(self.part(name + "_scale")).transpose(0, 2, 1).reshape(-1, self.heads, 1)
            x = x * sc
        return x


def attention(cache, q, table, lens, max_len, scale, window):
    """Outputs and log-sums [B][heads][dim], [B][heads] in 64 bits, and per output the sums
    that its tolerance is made of: a = sum p |v|, s = the largest |score| and x = the
    largest scale * k_scale * sum |q| |k| of its head."""
    B, heads, dim = q.shape
    k, v = cache.rows("k"), cache.rows("v")
    group = heads // cache.heads
    out, lse = np.zeros(q.shape), np.full((B, heads), -np.inf)
    a, s_top, x_top = np.zeros(q.shape), np.zeros((B, heads)), np.zeros((B, heads))
    for b in range(B):
        n = min(max(int(lens[b]), 0), max_len)
        t = np.arange(max(0, n - window) if window else 0, n)
        page = table[b][t // cache.page] if n else t
        t = t[(page >= 0) & (page < cache.pages)]
        if not len(t):
            continue
        at = table[b][t // cache.page].astype(np.int64) * cache.page + t % cache.page
        for h in range(heads):
            kk, vv = k[at, h // group], v[at, h // group]
            s = scale * (kk @ q[b, h])
            m = s.max()
            p = np.exp(s - m)
            l = p.sum()
            out[b, h], lse[b, h] = (p @ vv) / l, m + np.log(l)
            a[b, h] = (p @ np.abs(vv)) / l
            s_top[b, h] = np.abs(s).max()
            x_top[b, h] = abs(scale) * (np.abs(kk) @ np.abs(q[b, h])).max()
    return out, lse, a, s_top, x_top


def attention_bound(want, a, s_top, x_top, n, dim, kind, rows):
    """What the kernel's roundings add up to at most (first order, worst case), per output.

    Score: dim products and their sum in fp32, one rounding (2^-23, the matrix
    instructions may cut) each, then two products and the subtraction of m:
    d = (dim + 8) 2^-23 x + 6 2^-24 s, in the exponent.  It enters a weight and the sum of the
    weights: 2 d.  exp2: 2 units in the last place, twice.  The weight's rounding
    for the second product: half a step of what the output's type gets (16 or 24 bits; 11 for
    F16 caches, and 2^-32 of the maximum below their normal range).  Sums: n / 16 + 64 additions for l,
    n / 4 + 64 for o, half of the roundings' worst case each 2^-23.  The division and the output's rounding."""
    half_p = 2.0 ** -11 if kind == "f16" else {"bf16": 2.0 ** -16, "f16": 2.0 ** -16, "f32": 2.0 ** -24}[rows]
    d = (dim + 8) * 2.0 ** -23 * x_top + 6 * 2.0 ** -24 * s_top
    rel = 2 * d + 4 * 2.0 ** -23 + half_p + (n / 16 + 64 + n / 4 + 64) * 2.0 ** -23
    small = n * 2.0 ** -32 if kind == "f16" else 0.0
    vmax = 8.0 if kind == "f16" else 0.0
    return rel[..., None] * a * 1.01 + small * vmax + HALF[rows] * np.abs(want) * 1.01 + 2.0 ** -24 * (rows == "f16")


def ref(struct):
    return ctypes.byref(struct)


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream
