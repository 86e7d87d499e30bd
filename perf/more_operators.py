"""More operators of an autoregressive decoder, as measurable cases.

What a decoder with rotary positions, prompts of several tokens and a cache in
4 bits runs beside the operators of perf/operators.py.  Sizes are generic,
around the encoder's own (width 1024, heads of 128).  Floating types are named
f32, bf16 and f16; caches also hold int8, e4m3 (one fp32 scale for each (token,
head) row) and e2m1 (4-bit floats, two a byte, the even element in the low half;
each 32 elements of a row share the power of two 2^(byte - 127)).

A case is a dict with "op" and that operator's sizes:
  rope    n tokens: queries are rotated to their positions, keys are rotated and
          written into the cache with the values; cache "" is rows alone (one set
          of rows, out of place).  `rot` elements of a head turn, as pairs of
          neighbours (interleaved) or of halves.  What an 8-bit cache then holds is
          read back
  write4  n rows of keys and values into a 4-bit cache, and back
  attn4   one new token for each of `batch` sequences over a 4-bit cache
  prompt  up to `new` new tokens for each of `batch` sequences of up to `len`
          tokens, and rows of padding behind them; `ragged` counts spread over
          [1, new] and what came before over [0, len - new], one sequence in a
          batch of three or more is idle.  cap > 0: scores go through cap *
          tanh(s / cap); bias: less slope * distance; window: the last tokens only;
          docs: documents of that mean length, which do not see each other; prefix:
          so many tokens at a document's (or the sequence's) begin are seen by all
          of it
"""
import ctypes
import importlib.util
import math
import os

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
         "int8": torch.int8, "e4m3": torch.float8_e4m3fn, "e2m1": torch.uint8}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "int8": 1, "e4m3": 1, "e2m1": 0.5}
TOP = {"int8": 127.0, "e4m3": 448.0}
TINY = 2.0 ** -100          # rows or groups below this are written as zeros
GROUP = 32                  # elements of a 4-bit row that share their power of two
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    plain = {"cap": 0.0, "bias": False, "window": 0, "docs": 0, "prefix": 0}
    return [
        # a decoding step of 33 sequences: positions and cache write, latency
        {"name": "rope_step", "op": "rope", "n": 33, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "interleaved": False, "scaled": False, "far": 5000, "page": 16, "dtype": "bf16", "cache": "bf16"},
        # prefixes of a batch far into a long context, half of each head turns, 8-bit cache
        {"name": "rope_prefix", "op": "rope", "n": 8191, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 64,
         "interleaved": True, "scaled": True, "far": 1000000, "page": 64, "dtype": "bf16", "cache": "int8"},
        # rows alone, fp32 as the encoder computes, small heads
        {"name": "rope_rows", "op": "rope", "n": 4001, "heads": 16, "kv_heads": 16, "dim": 64, "rot": 64,
         "interleaved": False, "scaled": False, "far": 5000, "page": 16, "dtype": "f32", "cache": ""},
        # prefixes of a batch go into a 4-bit cache
        {"name": "write4_prefix", "op": "write4", "n": 8191, "heads": 8, "dim": 128, "page": 32, "dtype": "bf16"},
        # one long session over 4 bits: the cache's length has to fill the chip
        {"name": "attn4_session", "op": "attn4", "batch": 1, "len": 100003, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16", "ragged": False},
        # a serving batch of ragged lengths over 4 bits
        {"name": "attn4_batch", "op": "attn4", "batch": 96, "len": 6000, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 32, "dtype": "bf16", "ragged": True},
        # single tokens of a model that caps its scores and takes distance off them, with a window
        dict(plain, name="token_rules", op="prompt", batch=64, new=1, len=6000, heads=32, kv_heads=8, dim=128, page=32,
             dtype="bf16", cache="int8", ragged=True, cap=30.0, bias=True, window=2048),
        # five drafted tokens of each sequence are checked at once: few rows over long caches
        dict(plain, name="draft_check", op="prompt", batch=16, new=5, len=4000, heads=32, kv_heads=8, dim=128, page=16,
             dtype="bf16", cache="bf16", ragged=True),
        # the text of one utterance as a prompt, fp32 as the encoder computes, every head its own keys: latency
        dict(plain, name="prompt_clip", op="prompt", batch=1, new=417, len=417, heads=8, kv_heads=8, dim=128, page=16,
             dtype="f32", cache="bf16", ragged=False),
        # documents packed into one sequence, the head of each seen by all of it
        dict(plain, name="prompt_packed", op="prompt", batch=1, new=8191, len=8191, heads=16, kv_heads=4, dim=64, page=32,
             dtype="f16", cache="f16", ragged=False, docs=900, prefix=64),
        # a ragged batch of chunks behind what is cached in 4 bits: wide heads, cap and window
        dict(plain, name="prompt_chunks", op="prompt", batch=8, new=2000, len=5000, heads=16, kv_heads=4, dim=256, page=64,
             dtype="bf16", cache="e2m1", ragged=True, cap=50.0, window=1024),
        # one long prompt
        dict(plain, name="prompt_long", op="prompt", batch=1, new=8192, len=8192, heads=32, kv_heads=8, dim=128, page=64,
             dtype="bf16", cache="bf16", ragged=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("rope", "rope", "write4", "attn4", "attn4", "prompt", "prompt", "prompt", "prompt"))
    if op == "rope":
        kv = rng.choice((1, 2, 4, 8))
        dim = rng.choice((64, 128, 128, 256))
        return {"op": op, "n": _log_int(rng, 1, 8000), "heads": kv * rng.choice((1, 2, 4, 8)) if dim < 256 else kv,
                "kv_heads": kv, "dim": dim, "rot": rng.choice((dim, dim, dim // 2, dim // 4 * 3, 2 * rng.randint(1, dim // 2))),
                "interleaved": rng.random() < 0.5, "scaled": rng.random() < 0.5, "far": _log_int(rng, 100, 1000000),
                "page": rng.choice((16, 32, 64, 256)), "dtype": rng.choice(("f32", "bf16", "f16")),
                "cache": rng.choice(("", "bf16", "f16", "int8", "e4m3"))}
    if op == "write4":
        return {"op": op, "n": _log_int(rng, 1, 8000), "heads": rng.randint(1, 8), "dim": rng.choice((64, 128, 128, 256)),
                "page": rng.choice((16, 32, 64, 256)), "dtype": rng.choice(("f32", "bf16", "f16"))}
    kv = rng.choice((1, 2, 3, 4, 8))
    dim = rng.choice((64, 128, 128, 256))
    if op == "attn4":
        batch = _log_int(rng, 1, 128)
        most = max(2, min(100000, 100003 * 8 * 128 // (batch * kv * dim)))
        return {"op": op, "batch": batch, "len": _log_int(rng, 1, most), "heads": kv * rng.choice((1, 2, 4, 5, 8, 16)),
                "kv_heads": kv, "dim": dim, "page": rng.choice((16, 32, 64, 256)),
                "dtype": rng.choice(("f32", "bf16", "f16")), "ragged": rng.random() < 0.7}
    heads = kv * rng.choice((1, 2, 3, 4, 8))
    cache = rng.choice(("bf16", "bf16", "f16", "int8", "e4m3", "e2m1"))
    dtype = {"bf16": rng.choice(("bf16", "bf16", "f32")), "f16": "f16"}.get(cache, rng.choice(("f32", "bf16", "f16")))
    batch = _log_int(rng, 1, 24)
    new = rng.choice((1, _log_int(rng, 2, 16), _log_int(rng, 16, 4000), _log_int(rng, 16, 4000)))
    # scores of every query head within a quarter of the largest listed case's
    most = max(new, min(20000, 32 * 8192 * 8192 // 4 // (batch * heads * new)))
    while batch > 1 and batch * heads * new * new > 32 * 8192 * 8192 // 4:
        batch //= 2
    length = _log_int(rng, new, max(new + 1, min(most, 32 * 8192 * 8 // (batch * kv))))
    return {"op": op, "batch": batch, "new": new, "len": length, "heads": heads, "kv_heads": kv, "dim": dim,
            "page": rng.choice((16, 32, 64, 256)), "dtype": dtype, "cache": cache, "ragged": rng.random() < 0.6,
            "cap": rng.choice((0.0, 0.0, 20.0, 50.0)), "bias": rng.random() < 0.3,
            "window": rng.choice((0, 0, 0, _log_int(rng, 1, max(2, length)))),
            "docs": rng.choice((0, 0, 0, _log_int(rng, 2, max(3, length)))),
            "prefix": rng.choice((0, 0, 0, _log_int(rng, 1, max(2, length))))}


# ---- inputs ------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device="cuda:0")
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _normal(g, shape, sd=1.0, mean=0.0):
    return torch.randn(shape, generator=g, device="cuda:0") * sd + mean


def _randint(g, lo, hi, shape, dtype):
    return torch.randint(lo, hi, shape, generator=g, device="cuda:0", dtype=dtype)


def _activations(g, rows, d, dtype):
    """Rows of projected keys or values: a few channels are much larger than the rest."""
    x = _normal(g, (rows, d))
    big = _randint(g, 0, d, (max(1, d // 128),), torch.int64)
    x[:, big] *= 8.0
    return x.to(TYPES[dtype])


def _cache(g, case, kind, pages, heads, filled):
    """k, v [pages][heads][page][dim] (e2m1: [dim / 2] bytes) and their scales."""
    page, dim = case["page"], case["dim"]
    shape = (pages, heads, page, dim // 2 if kind == "e2m1" else dim)
    got = {}
    for name in ("k", "v"):
        if not filled:
            got[name] = torch.zeros(shape, device="cuda:0", dtype=TYPES[kind])
        elif kind == "int8":
            got[name] = _randint(g, -127, 128, shape, torch.int8)
        elif kind == "e2m1":
            got[name] = _randint(g, 0, 256, shape, torch.uint8)
        elif kind == "e4m3":
            got[name] = (_normal(g, shape, 120.0)).clamp_(-448.0, 448.0).to(TYPES[kind])
        else:
            got[name] = _normal(g, shape).to(TYPES[kind])
        if kind in TOP:
            top = torch.rand(shape[:3], generator=g, device="cuda:0") * 3.0 + 1.0
            got[name + "_scale"] = (top / TOP[kind]) if filled else torch.zeros(shape[:3], device="cuda:0")
        elif kind == "e2m1":
            groups = shape[:3] + (dim // GROUP,)
            got[name + "_scale"] = (_randint(g, 124, 127, groups, torch.uint8) if filled
                                    else torch.zeros(groups, device="cuda:0", dtype=torch.uint8))
    return got


def _slots(g, n, pages, page):
    """Distinct slots of n tokens, whole pages one after another, 1 row in 32 padding."""
    order = torch.randperm(pages, generator=g, device="cuda:0")
    s = (order[:, None] * page + torch.arange(page, device="cuda:0")).reshape(-1)[:n]
    pad = torch.rand((n,), generator=g, device="cuda:0") < 1.0 / 32
    return torch.where(pad, -1, s).to(torch.int32)


def _freqs(case):
    """Frequencies of the turning pairs, for scaled ones a long context's: low ones 8 times lower."""
    i = torch.arange(0, case["rot"], 2, dtype=torch.float64)
    f = 10000.0 ** (-i / case["rot"])
    if case["scaled"]:
        turns = 8192.0 * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        f = f * (keep + (1.0 - keep) / 8.0)
    return f.float().to("cuda:0")


def _paged(s, g, batch, most, page, kind, heads):
    """Lengths are there: the sequences' pages, in any order, absent ones -1."""
    per = max(1, (most + page - 1) // page)
    s["pages"] = batch * per + 1
    table = torch.randperm(batch * per, generator=g, device="cuda:0").reshape(batch, per).to(torch.int32)
    used = torch.arange(per, device="cuda:0") * page < s["lens"][:, None]
    s["table"] = torch.where(used, table, -1).to(torch.int32).contiguous()
    s.update(_cache(g, s["case"], kind, s["pages"], heads, True))


def _prepare_prompt(s, g, case):
    b, new, most = case["batch"], case["new"], case["len"]
    counts = torch.full((b,), new, device="cuda:0", dtype=torch.int32)
    before = torch.full((b,), most - new, device="cuda:0", dtype=torch.int32)
    if case["ragged"]:
        # as many rows whatever the seed: counts spread evenly, in any order, one sequence idle
        counts = torch.linspace(new, 1, b, device="cuda:0").round().to(torch.int32)
        if b > 2:
            counts[-1] = 0
        before = _randint(g, 0, most - new + 1, (b,), torch.int32)
        before[:1] = most - new
        order = torch.randperm(b, generator=g, device="cuda:0")
        counts, before = counts[order], before[order]
    s["lens"] = counts + before
    s["starts"] = torch.cat([torch.zeros(1, device="cuda:0", dtype=torch.int32), counts.cumsum(0).to(torch.int32)])
    live = int(s["starts"][-1])
    s["rows"] = live + -live % 16              # rows for a fixed launch: the last ones are padding
    _paged(s, g, b, most, case["page"], case["cache"], case["kv_heads"])
    wide = case["heads"] * case["dim"]
    s["q"] = _normal(g, (s["rows"], wide)).to(TYPES[case["dtype"]])
    s["out"] = torch.zeros_like(s["q"])
    s["scale"] = 1.0 / math.sqrt(case["dim"])
    h = torch.arange(1, case["heads"] + 1, device="cuda:0", dtype=torch.float32)
    s["slopes"] = torch.exp2(-8.0 * h / case["heads"]) if case["bias"] else None
    # each live row's sequence and position
    s["row_b"] = torch.repeat_interleave(torch.arange(b, device="cuda:0"), counts.long())
    s["row_p"] = (torch.arange(live, device="cuda:0") - s["starts"][s["row_b"]].long()
                  + before[s["row_b"]].long())
    s["first"] = s["until"] = None
    if case["docs"] or case["prefix"]:
        t = torch.arange(most, device="cuda:0")
        begins = torch.zeros((b, most), device="cuda:0", dtype=torch.bool)
        if case["docs"]:
            begins = torch.rand((b, most), generator=g, device="cuda:0") < 1.0 / case["docs"]
        begin = torch.where(begins, t, 0).cummax(1).values
        first = torch.zeros((s["rows"],), device="cuda:0", dtype=torch.int32)
        first[:live] = begin[s["row_b"], s["row_p"]].to(torch.int32)
        if case["docs"]:
            s["first"] = first
        if case["prefix"]:       # within the document
            later = torch.where(begins, t, most).flip(1).cummin(1).values.flip(1)
            later = torch.cat([later[:, 1:], torch.full((b, 1), most, device="cuda:0")], 1)[s["row_b"], s["row_p"]]
            s["until"] = torch.zeros_like(first)
            s["until"][:live] = torch.minimum(first[:live].long() + case["prefix"], later).to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": dict(case), "kept": {}}
    op = case["op"]
    if op in ("rope", "write4"):
        n, dim, page = case["n"], case["dim"], case["page"]
        kind = "e2m1" if op == "write4" else case["cache"]
        heads = case["heads"] if op == "write4" else case["kv_heads"]
        pages = (n + page - 1) // page + 3
        s["pages"] = pages
        s["slots"] = _slots(g, n, pages, page)
        if kind:         # one page behind the cache's last: where the plain form puts padding rows
            s.update(_cache(g, case, kind, pages + 1, heads, False))
            for name in ("new_k", "new_v"):
                s[name] = _activations(g, n, heads * dim, case["dtype"])
        if op == "rope":
            s["x"] = _activations(g, n, case["heads"] * dim, case["dtype"])
            s["y"] = torch.empty_like(s["x"])
            s["pos"] = _randint(g, 0, case["far"], (n,), torch.int32)
            s["freqs"] = _freqs(case)
            s["mag"] = 0.1 * math.log(8.0) + 1.0 if case["scaled"] else 1.0
        if kind in TOP or kind == "e2m1":
            s["out_k"] = torch.zeros((n, heads * dim), device="cuda:0", dtype=TYPES[case["dtype"]])
            s["out_v"] = torch.zeros_like(s["out_k"])
    elif op == "attn4":
        b, most = case["batch"], case["len"]
        lens = torch.full((b,), most, device="cuda:0", dtype=torch.int32)
        if case["ragged"]:
            lens = _randint(g, 0, most + 1, (b,), torch.int32)
            lens[:1], lens[1:2], lens[2:3] = most, 0, 1
        s["lens"] = lens
        _paged(s, g, b, most, case["page"], "e2m1", case["kv_heads"])
        s["q"] = _normal(g, (b, case["heads"] * case["dim"])).to(TYPES[case["dtype"]])
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(case["dim"])
    else:
        _prepare_prompt(s, g, case)
    return s


# ---- the plain forms ---------------------------------------------------------

def _rotated(s, x, heads):
    """x [n][heads * dim] in fp32, turned; angles in 64 bits."""
    case = s["case"]
    n, dim, rot = case["n"], case["dim"], case["rot"]
    x = x.float().reshape(n, heads, dim)
    angle = s["pos"].double()[:, None] * s["freqs"].double()
    c = (torch.cos(angle) * s["mag"]).float()[:, None]
    z = (torch.sin(angle) * s["mag"]).float()[:, None]
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack([a * c - b * z, b * c + a * z], -1).reshape(n, heads, rot)
    else:
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        turned = torch.cat([a * c - b * z, b * c + a * z], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _stored(s, name, x, kind):
    """x [n][heads][dim] in fp32 into the cache's slots."""
    page = s["case"]["page"]
    slot = torch.where(s["slots"] < 0, s["pages"] * page, s["slots"]).long()
    at, off = slot // page, slot % page
    if kind in TOP:
        amax = x.abs().amax(-1)
        zero = amax < TINY
        inv = torch.where(zero, 0.0, TOP[kind] / amax)
        s[name + "_scale"][at, :, off] = torch.where(zero, 0.0, amax / TOP[kind])
        x = (x * inv[..., None]).clamp(-TOP[kind], TOP[kind])
    if kind == "int8":
        x = x.round()
    if kind == "e2m1":
        n, heads, dim = x.shape
        x = x.reshape(n, heads, dim // GROUP, GROUP)
        amax = x.abs().amax(-1)
        zero = amax < TINY
        _, e = torch.frexp(torch.where(zero, 1.0, amax))      # amax = m 2^e, m in [1/2, 1)
        e = e - 3
        e = torch.where(amax > torch.ldexp(torch.full_like(amax, 7.0), e), e + 1, e).clamp_max(125)
        y = torch.where(zero[..., None], 0.0, torch.ldexp(x, -e[..., None]))
        size = y.abs()
        # ties to the even code: borders that round down are passed from above only
        code = ((size > 0.25).int() + (size >= 0.75) + (size > 1.25) + (size >= 1.75) + (size > 2.5) + (size >= 3.5)
                + (size > 5.0))
        code = (code + 8 * (y < 0.0)).to(torch.uint8).reshape(n, heads, dim // 2, 2)
        s[name + "_scale"][at, :, off] = torch.where(zero, 0, e + 127).to(torch.uint8)
        s[name][at, :, off] = code[..., 0] + 16 * code[..., 1]
    elif kind == "e4m3":     # indexed stores go by bytes
        s[name].view(torch.uint8)[at, :, off] = x.to(TYPES["e4m3"]).view(torch.uint8)
    else:
        s[name][at, :, off] = x.to(TYPES[kind])


def _levels():
    return torch.tensor(LEVELS + tuple(-v for v in LEVELS), device="cuda:0")


def _held(s, name, pick, kind):
    """Cache entries named by the index `pick` in fp32, the head's elements last."""
    if kind == "e4m3":
        return s[name].view(torch.uint8)[pick].view(TYPES[kind]).float() * s[name + "_scale"][pick][..., None]
    if kind == "int8":
        return s[name][pick].float() * s[name + "_scale"][pick][..., None]
    if kind != "e2m1":
        return s[name][pick].float()
    b = s[name][pick]
    x = _levels()[torch.stack([b & 15, b >> 4], -1).long()]
    e = s[name + "_scale"][pick].float() - 127.0
    x = x.reshape(b.shape[:-1] + (-1, GROUP)) * torch.exp2(e)[..., None]
    return x.reshape(b.shape[:-1] + (-1,))


def _back(s, kind):
    case = s["case"]
    slot = s["slots"].long().clamp_min(0)
    there = (s["slots"] >= 0)[:, None, None]
    pick = (slot // case["page"], slice(None), slot % case["page"])
    return [torch.where(there, _held(s, name, pick, kind), 0.0).reshape(case["n"], -1).to(TYPES[case["dtype"]])
            for name in ("k", "v")]


def _plain_rope(s):
    case = s["case"]
    kind = case["cache"]
    y = _rotated(s, s["x"], case["heads"]).reshape(s["x"].shape).to(s["x"].dtype)
    if not kind:
        return y
    _stored(s, "k", _rotated(s, s["new_k"], case["kv_heads"]), kind)
    _stored(s, "v", s["new_v"].float().reshape(case["n"], case["kv_heads"], case["dim"]), kind)
    if kind in TOP:
        return [y] + _back(s, kind)
    return [y, s["k"][:s["pages"]], s["v"][:s["pages"]]]


def _plain_write4(s):
    case = s["case"]
    shape = (case["n"], case["heads"], case["dim"])
    _stored(s, "k", s["new_k"].float().reshape(shape), "e2m1")
    _stored(s, "v", s["new_v"].float().reshape(shape), "e2m1")
    return _back(s, "e2m1")


def _sides(s, kind):
    """Keys and values [batch][kv heads][tokens][dim] of the page tables."""
    table = s["table"].long().clamp_min(0)
    return [(lambda x: x.transpose(1, 2).reshape(x.shape[0], x.shape[2], -1, x.shape[-1]))(_held(s, name, table, kind))
            for name in ("k", "v")]


def _softmax_times(score, seen, v):
    """Softmax over the last axis of what is seen, times v [..][tokens][dim]; zeros where nothing is."""
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p / torch.where(total == 0.0, 1.0, total), v)


def _plain_attn4(s):
    case = s["case"]
    b, kv, dim = case["batch"], case["kv_heads"], case["dim"]
    k, v = _sides(s, "e2m1")
    q = s["q"].float().reshape(b, kv, -1, dim)
    score = torch.matmul(q, k.transpose(2, 3).contiguous()) * s["scale"]
    seen = torch.arange(k.shape[2], device="cuda:0") < s["lens"][:, None, None, None]
    return _softmax_times(score, seen, v).reshape(s["q"].shape).to(s["q"].dtype)


def _plain_prompt(s):
    case = s["case"]
    b, kv, dim, new = case["batch"], case["kv_heads"], case["dim"], case["new"]
    group = case["heads"] // kv
    k, v = _sides(s, case["cache"])
    row_b = s["row_b"]
    live = row_b.shape[0]
    row_i = torch.arange(live, device="cuda:0") - s["starts"].long()[row_b]
    q = torch.zeros((b, new, kv, group, dim), device="cuda:0")
    q[row_b, row_i] = s["q"][:live].float().reshape(-1, kv, group, dim)
    q = q.permute(0, 2, 3, 1, 4).reshape(b, kv, group * new, dim).contiguous()
    score = torch.matmul(q, k.transpose(2, 3).contiguous()).reshape(b, kv, group, new, -1)
    score *= s["scale"]
    if case["cap"]:
        score = case["cap"] * torch.tanh(score / case["cap"])
    place = torch.zeros((3, b, new), device="cuda:0", dtype=torch.int64)     # position, first seen, first not seen
    p = s["row_p"]
    first = s["first"][:live].long() if s["first"] is not None else torch.zeros_like(p)
    if case["window"]:
        first = torch.maximum(first, p - case["window"] + 1)
    until = p + 1 if s["until"] is None else torch.maximum(p + 1, s["until"][:live].long())
    place[:, row_b, row_i] = torch.stack([p, first, torch.minimum(until, s["lens"].long()[row_b])])
    place = place.reshape(3, b, 1, 1, new, 1)
    t = torch.arange(k.shape[2], device="cuda:0")
    if s["slopes"] is not None:
        score -= s["slopes"].reshape(1, kv, group, 1, 1) * (place[0] - t).abs().float()
    seen = (t >= place[1]) & (t < place[2])
    out = _softmax_times(score.reshape(b, kv, group * new, -1),
                         seen.expand(b, 1, group, new, t.shape[0]).reshape(b, 1, group * new, -1), v)
    out = out.reshape(b, kv, group, new, dim).permute(0, 3, 1, 2, 4)
    rows = torch.zeros_like(s["q"])
    rows[:live] = out[row_b, row_i].reshape(live, -1).to(rows.dtype)
    return rows


def _plain(s):
    return {"rope": _plain_rope, "write4": _plain_write4, "attn4": _plain_attn4, "prompt": _plain_prompt}[s["case"]["op"]](s)


# ---- the framework's calls ---------------------------------------------------

_bound = []


def _pk():
    if not _bound:
        path = os.path.join(os.getcwd(), "parakeet-unified-en-0.6b-c_amd", "pk_gpu_ctypes.py")
        spec = importlib.util.spec_from_file_location("pk_gpu_ctypes", path)
        pk = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(pk)
        pk.call("pk_gpu_init", 0)
        _bound.append(pk)
    return _bound[0]


def _kind(pk, name):
    return {"f32": pk.F32, "f16": pk.F16, "bf16": pk.BF16, "int8": pk.I8, "e4m3": pk.E4M3, "e2m1": pk.E2M1}[name]


def _at(t):
    return t.data_ptr() if t is not None else None


def _own_cache(pk, s, kind, heads):
    """The cache's description: made once, as a program that holds the cache does."""
    kept = s["kept"]
    if "cache" not in kept:
        case = s["case"]
        kept["cache"] = pk.KvCache(s["k"].data_ptr(), s["v"].data_ptr(), _at(s.get("k_scale")), _at(s.get("v_scale")),
                                   _kind(pk, kind), s["pages"], case["page"], heads, case["dim"])
        kept["cache_p"] = ctypes.byref(kept["cache"])
    return kept["cache_p"]


def _own_back(pk, s, cache, wide, stream):
    pk.call("pk_gpu_kv_read_dev", cache, _kind(pk, s["case"]["dtype"]), s["slots"].data_ptr(), s["case"]["n"],
            s["out_k"].data_ptr(), wide, s["out_v"].data_ptr(), wide, stream)
    return [s["out_k"], s["out_v"]]


def _own_rope(pk, s, stream):
    case, kept = s["case"], s["kept"]
    if "rope" not in kept:
        kept["rope"] = pk.Rope(s["freqs"].data_ptr(), s["mag"], case["rot"], int(case["interleaved"]))
        kept["rope_p"] = ctypes.byref(kept["rope"])
    kind, kv, dim, n = case["cache"], case["kv_heads"], case["dim"], case["n"]
    wide, dtype = case["heads"] * dim, _kind(pk, case["dtype"])
    if not kind:
        pk.call("pk_gpu_rope_dev", kept["rope_p"], dtype, s["x"].data_ptr(), wide, case["heads"], dim,
                s["pos"].data_ptr(), n, s["y"].data_ptr(), wide, stream)
        return s["y"]
    cache = _own_cache(pk, s, kind, kv)
    pk.call("pk_gpu_rope_kv_write_dev", kept["rope_p"], cache, dtype, s["x"].data_ptr(), wide, case["heads"],
            s["y"].data_ptr(), wide, s["new_k"].data_ptr(), kv * dim, s["new_v"].data_ptr(), kv * dim,
            s["pos"].data_ptr(), s["slots"].data_ptr(), n, stream)
    if kind in TOP:
        return [s["y"]] + _own_back(pk, s, cache, kv * dim, stream)
    return [s["y"], s["k"][:s["pages"]], s["v"][:s["pages"]]]


def _own_write4(pk, s, stream):
    case = s["case"]
    wide = case["heads"] * case["dim"]
    cache = _own_cache(pk, s, "e2m1", case["heads"])
    pk.call("pk_gpu_kv_write_dev", cache, _kind(pk, case["dtype"]), s["new_k"].data_ptr(), wide,
            s["new_v"].data_ptr(), wide, s["slots"].data_ptr(), case["n"], stream)
    return _own_back(pk, s, cache, wide, stream)


def _own_attn4(pk, s, stream):
    case, kept = s["case"], s["kept"]
    cache = _own_cache(pk, s, "e2m1", case["kv_heads"])
    wide = case["heads"] * case["dim"]
    if "floats" not in kept:
        kept["floats"] = pk.load().pk_gpu_paged_attention_ws_floats(cache, case["batch"], case["heads"], case["len"], 0)
        kept["ws"] = torch.empty((max(1, kept["floats"]),), device="cuda:0")
    pk.call("pk_gpu_paged_attention_dev", cache, _kind(pk, case["dtype"]), s["q"].data_ptr(), wide, case["heads"],
            s["table"].data_ptr(), s["table"].shape[1], s["lens"].data_ptr(), case["batch"], case["len"],
            s["scale"], 0, s["out"].data_ptr(), wide, None, kept["ws"].data_ptr(), kept["floats"], stream)
    return s["out"]


def _own_prompt(pk, s, stream):
    case, kept = s["case"], s["kept"]
    cache = _own_cache(pk, s, case["cache"], case["kv_heads"])
    wide = case["heads"] * case["dim"]
    if "floats" not in kept:
        kept["rules"] = pk.AttentionRules(s["scale"], case["cap"], _at(s["slopes"]), case["window"], _at(s["first"]),
                                          _at(s["until"]))
        kept["rules_p"] = ctypes.byref(kept["rules"])
        kept["floats"] = pk.load().pk_gpu_prompt_attention_ws_floats(cache, case["batch"], s["rows"], case["heads"],
                                                                     case["new"], case["len"], case["window"])
        kept["ws"] = torch.empty((max(1, kept["floats"]),), device="cuda:0")
    pk.call("pk_gpu_prompt_attention_dev", cache, _kind(pk, case["dtype"]), s["q"].data_ptr(), wide, case["heads"],
            s["table"].data_ptr(), s["table"].shape[1], s["lens"].data_ptr(), s["starts"].data_ptr(), case["batch"],
            s["rows"], case["new"], case["len"], kept["rules_p"], s["out"].data_ptr(), wide, None,
            kept["ws"].data_ptr(), kept["floats"], stream)
    return s["out"]


def _own(s):
    pk = _pk()
    stream = torch.cuda.current_stream().cuda_stream
    return {"rope": _own_rope, "write4": _own_write4, "attn4": _own_attn4, "prompt": _own_prompt}[s["case"]["op"]](pk, s, stream)


def run(state):
    return _own(state) if own else _plain(state)


# ---- work and exact values ---------------------------------------------------

def _row_bytes(kind, dim):
    return dim * SIZE[kind] + (4 if kind in TOP else dim // GROUP if kind == "e2m1" else 0)


def _pairs(case):
    """Query-token pairs that a case's rows see, on average over what is drawn."""
    new, most = case["new"], case["len"]
    n = (new + 1) / 2 if case["ragged"] else new
    before = (most - new) / 2 if case["ragged"] else most - new
    reach = case["window"] or most
    seen = before + (n + 1) / 2                       # each row's, on average
    if reach < before + n:
        seen = reach if reach <= before else (reach - before) / n * (before + reach) / 2 + (before + n - reach) / n * reach
    return case["batch"] * n * min(seen, reach, case["docs"] or most)


def work(case):
    op, size, dim = case["op"], SIZE[case["dtype"]], case["dim"]
    if op == "rope":
        rows = 2 * case["n"] * case["heads"] * dim * size + 4 * case["n"] + 2 * case["rot"]
        if case["cache"]:
            held = 2 * case["n"] * case["kv_heads"] * _row_bytes(case["cache"], dim)
            given = 2 * case["n"] * case["kv_heads"] * dim * size
            rows += held + given + 4 * case["n"] + (held + given if case["cache"] in TOP else 0)
        return {"bytes": rows, "flops": 0}
    if op == "write4":
        rows = 2 * case["n"] * case["heads"]
        return {"bytes": 2 * rows * (_row_bytes("e2m1", dim) + dim * size) + 8 * case["n"], "flops": 0}
    if op == "attn4":
        t = case["batch"] * case["len"] * (0.5 if case["ragged"] else 1.0)
        return {"bytes": 2 * t * case["kv_heads"] * _row_bytes("e2m1", dim) + 2 * case["batch"] * case["heads"] * dim * size,
                "flops": 4 * t * case["heads"] * dim}
    n = case["batch"] * ((case["new"] + 1) / 2 if case["ragged"] else case["new"])
    length = case["len"] * (0.5 if case["ragged"] else 1.0)
    if case["window"]:
        length = min(length, case["window"] + n / case["batch"])
    t = case["batch"] * length
    return {"bytes": 2 * t * case["kv_heads"] * _row_bytes(case["cache"], dim) + 2 * n * case["heads"] * dim * size,
            "flops": 4 * _pairs(case) * case["heads"] * dim}


def _value(s, name, kind, pages):
    """[tokens][heads][dim] in 64 bits that a list of pages holds."""
    x = s[name][pages] if kind != "e4m3" else s[name].view(torch.uint8)[pages].view(TYPES[kind])
    if kind == "e2m1":
        low, high = (x & 15).int(), (x >> 4).int()
        x = torch.empty(x.shape[:-1] + (2 * x.shape[-1],), device="cuda:0", dtype=torch.float64)
        for part, code in ((0, low), (1, high)):
            e, m = code >> 1 & 3, code & 1
            size = torch.where(e > 0, torch.ldexp(1.0 + 0.5 * m.double(), e - 1), 0.5 * m.double())
            x[..., part::2] = torch.where(code >= 8, -size, size)
        x = x * torch.ldexp(torch.ones((), device="cuda:0", dtype=torch.float64),
                            s[name + "_scale"][pages].int() - 127).repeat_interleave(GROUP, -1)
    else:
        x = x.double()
        if kind in TOP:
            x = x * s[name + "_scale"][pages].double().unsqueeze(-1)
    return x.transpose(1, 2).reshape(-1, x.shape[1], x.shape[3])


def _near(x, kind):
    """In 64 bits: what the codes of the last axis's rows stand for."""
    if kind == "e2m1":
        shape = x.shape
        x = x.reshape(shape[:-1] + (shape[-1] // GROUP, GROUP))
        big = x.abs().amax(-1, keepdim=True)
        u = torch.exp2(torch.ceil(torch.log2(big.clamp_min(1e-300) / 7.0)))
        u = torch.where(big > 7.0 * u, 2.0 * u, torch.where(big <= 3.5 * u, 0.5 * u, u))
        y = (x / u).abs()
        step = torch.exp2(torch.floor(torch.log2(y.clamp_min(1.0))) - 1.0)
        y = (torch.round(y / step) * step).clamp_max(6.0)
        return (torch.where(big < TINY, torch.zeros_like(x), torch.sign(x) * y * u)).reshape(shape)
    if kind not in TOP:
        return x
    big = x.abs().amax(-1, keepdim=True)
    u = big / TOP[kind]
    y = torch.where(big < TINY, torch.zeros_like(x), x / u.clamp_min(1e-300))
    if kind == "int8":
        return y.round() * u
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3.0)
    return torch.round(y / step) * step * u


def _exact_turn(s, x, heads):
    case = s["case"]
    half = case["rot"] // 2
    x = x.double().reshape(case["n"], heads, case["dim"])
    at = torch.arange(half, device="cuda:0")
    at = (2 * at, 2 * at + 1) if case["interleaved"] else (at, at + half)
    z = torch.complex(x[..., at[0]], x[..., at[1]])
    turn = torch.polar(torch.full((case["n"], 1, half), float(torch.tensor(s["mag"]).float()), device="cuda:0",
                                  dtype=torch.float64), torch.outer(s["pos"].double(), s["freqs"].double())[:, None])
    z = z * turn
    y = x.clone()
    y[..., at[0]], y[..., at[1]] = z.real, z.imag
    return y


def _exact_rows(s, kind, k, v):
    """What comes back of keys and values [n][heads][dim]: the rows, or the cache's own arrays."""
    case = s["case"]
    if kind in TOP or kind == "e2m1":
        keep = (s["slots"] >= 0).double()[:, None]
        return [_near(x, kind).reshape(case["n"], -1) * keep for x in (k, v)]
    got = []
    there = s["slots"] >= 0
    for x in (k, v):
        flat = torch.zeros((s["pages"] * case["page"],) + x.shape[1:], device="cuda:0", dtype=torch.float64)
        flat[s["slots"][there].long()] = x[there]
        got.append(flat.reshape(s["pages"], case["page"], x.shape[1], x.shape[2]).transpose(1, 2).contiguous())
    return got


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        y = _exact_turn(s, s["x"], case["heads"]).reshape(case["n"], -1)
        if not case["cache"]:
            return y
        shape = (case["n"], case["kv_heads"], case["dim"])
        return [y] + _exact_rows(s, case["cache"], _exact_turn(s, s["new_k"], case["kv_heads"]),
                                 s["new_v"].double().reshape(shape))
    if op == "write4":
        shape = (case["n"], case["heads"], case["dim"])
        return _exact_rows(s, "e2m1", s["new_k"].double().reshape(shape), s["new_v"].double().reshape(shape))
    kind = "e2m1" if op == "attn4" else case["cache"]
    kv, dim, heads = case["kv_heads"], case["dim"], case["heads"]
    group = heads // kv
    out = torch.zeros((s["q"].shape[0], heads, dim), device="cuda:0", dtype=torch.float64)
    lens = s["lens"].tolist()
    starts = s["starts"].tolist() if op == "prompt" else list(range(case["batch"] + 1))
    for b, n in enumerate(lens):
        rows = slice(starts[b], starts[b + 1])
        if not n or rows.start == rows.stop:
            continue
        pages = s["table"][b, :(n - 1) // case["page"] + 1].long()
        k, v = _value(s, "k", kind, pages)[:n], _value(s, "v", kind, pages)[:n]
        t = torch.arange(n, device="cuda:0")
        p = torch.arange(n - (rows.stop - rows.start), n, device="cuda:0").unsqueeze(1)
        hidden = t > p
        if op == "prompt":
            if s["until"] is not None:
                hidden &= t >= s["until"][rows].unsqueeze(1)
            if s["first"] is not None:
                hidden |= t < s["first"][rows].unsqueeze(1)
            if case["window"]:
                hidden |= t <= p - case["window"]
        for h in range(heads):
            w = s["q"][rows].double().reshape(-1, heads, dim)[:, h] @ k[:, h // group].t().contiguous() / math.sqrt(dim)
            if op == "prompt" and case["cap"]:
                w = torch.tanh(w / case["cap"]) * case["cap"]
            if op == "prompt" and case["bias"]:
                w -= s["slopes"][h].double() * (t - p).abs()
            w = torch.softmax(w.masked_fill(hidden, -torch.inf), -1)
            out[rows, h] = torch.nan_to_num(w, nan=0.0) @ v[:, h // group]
    return out.reshape(s["q"].shape)
