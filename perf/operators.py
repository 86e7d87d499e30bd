"""The operators of an autoregressive decoder's step, as measurable cases.

One block's step over the encoder's frames normalises its rows, projects
them, writes the new keys and values into a paged cache and attends over it.
Sizes are generic, around the encoder's own (width 1024, feed-forward 4096,
heads of 128).  Floating types are named f32, bf16 and f16; caches also hold
int8 and e4m3 codes with one fp32 scale for each (token, head) row.

A case is a dict with "op" and that operator's sizes:
  write  n rows of keys and values go into the cache's slots and are read
         back from them as a program that moves a prefix does (what the
         codes stand for is the output); some rows are padding (slot -1)
  read   n rows of a cache, read back
  attn   one new token for each of `batch` sequences of up to `len` tokens
         attends over the paged cache; `ragged` lengths spread over
         [0, len], otherwise all are `len`; `window` > 0 keeps the last
         `window` tokens
  norm   root-mean-square norm of rows + residual; the sum is stored too
  gemm   int8 rows with row scales x int8 weights, bias, activation or
         residual in the epilogue
  proj   norm with an int8 output, then gemm on its codes
"""
import ctypes
import importlib.util
import math
import os

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16,
         "int8": torch.int8, "e4m3": torch.float8_e4m3fn}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "int8": 1, "e4m3": 1}
TOP = {"int8": 127.0, "e4m3": 448.0}
TINY = 2.0 ** -100          # rows below this are written as zeros
EPS = 1e-5


def listed():
    return [
        # a decoding step of 32 sequences puts its new token into an int8 cache: latency
        {"name": "write_step", "op": "write", "n": 32, "heads": 8, "dim": 128, "page": 16,
         "dtype": "f32", "cache": "int8"},
        # prefixes of a batch, 8191 tokens, go into an 8-bit floating cache
        {"name": "write_prefix", "op": "write", "n": 8191, "heads": 8, "dim": 128, "page": 64,
         "dtype": "bf16", "cache": "e4m3"},
        # the cached prefixes of a batch come back for a program that moves them
        {"name": "read_prefix", "op": "read", "n": 20011, "heads": 8, "dim": 128, "page": 32,
         "dtype": "bf16", "cache": "int8"},
        # one utterance, every head its own keys, fp32 as the encoder computes: latency
        {"name": "attn_clip", "op": "attn", "batch": 1, "len": 417, "window": 0, "ragged": False,
         "heads": 8, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "f32", "cache": "int8"},
        # one long session: the cache's length has to fill the chip
        {"name": "attn_session", "op": "attn", "batch": 1, "len": 100003, "window": 0, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "dtype": "bf16", "cache": "bf16"},
        # a serving batch of ragged lengths over a quantised cache
        {"name": "attn_batch", "op": "attn", "batch": 96, "len": 6000, "window": 0, "ragged": True,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 32, "dtype": "bf16", "cache": "int8"},
        # many sequences, few wide shared heads, the last 1024 tokens of each
        {"name": "attn_window", "op": "attn", "batch": 160, "len": 5000, "window": 1024, "ragged": True,
         "heads": 16, "kv_heads": 1, "dim": 256, "page": 128, "dtype": "f16", "cache": "e4m3"},
        # the norm of a decoding step: latency
        {"name": "norm_step", "op": "norm", "rows": 33, "d": 1024, "dtype": "f32"},
        # the norm over a batch's prefixes
        {"name": "norm_prefix", "op": "norm", "rows": 8192, "d": 4096, "dtype": "bf16"},
        # up projection of a decoding step, norm included: the weights' bytes count
        {"name": "proj_step", "op": "proj", "m": 33, "n": 4096, "k": 1024, "dtype": "f32",
         "epilogue": "swish"},
        # the same over prefixes, odd row count
        {"name": "proj_prefix", "op": "proj", "m": 4001, "n": 4096, "k": 1024, "dtype": "bf16",
         "epilogue": "swish"},
        # a wide model's down projection over a batch's prefixes, into the residual stream
        {"name": "gemm_prefix", "op": "gemm", "m": 8192, "n": 4096, "k": 8192, "dtype": "bf16",
         "epilogue": "residual"},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("write", "read", "attn", "attn", "attn", "norm", "gemm", "proj"))
    if op in ("write", "read"):
        cache = rng.choice(("int8", "int8", "e4m3", "bf16", "f16"))
        return {"op": op, "n": _log_int(rng, 1, 8192 if op == "write" else 20000),
                "heads": rng.randint(1, 8), "dim": rng.choice((64, 128, 128, 256)),
                "page": rng.choice((16, 32, 64, 256)),
                "dtype": rng.choice(("f32", "bf16", "f16")), "cache": cache}
    if op == "attn":
        kv = rng.choice((1, 2, 3, 4, 8))
        group = rng.choice((1, 2, 4, 5, 8, 16))
        dim = rng.choice((64, 128, 128, 256))
        cache = rng.choice(("int8", "int8", "e4m3", "bf16", "f16"))
        dtype = {"bf16": rng.choice(("bf16", "f32")), "f16": "f16"}.get(cache, rng.choice(("f32", "bf16", "f16")))
        batch = _log_int(rng, 1, 128)
        most = max(2, min(100000, 100003 * 8 * 128 // (batch * kv * dim)))
        length = _log_int(rng, 1, most)
        window = rng.choice((0, 0, 0, _log_int(rng, 1, max(2, length))))
        return {"op": op, "batch": batch, "len": length, "window": window, "ragged": rng.random() < 0.7,
                "heads": kv * group, "kv_heads": kv, "dim": dim, "page": rng.choice((16, 32, 64, 256)),
                "dtype": dtype, "cache": cache}
    if op == "norm":
        return {"op": op, "rows": _log_int(rng, 1, 8192), "d": _log_int(rng, 64, 4096),
                "dtype": rng.choice(("f32", "bf16", "f16"))}
    if op == "gemm":
        return {"op": op, "m": _log_int(rng, 1, 8192), "n": _log_int(rng, 64, 4096), "k": _log_int(rng, 64, 8192),
                "dtype": rng.choice(("f32", "bf16", "f16")), "epilogue": rng.choice(("none", "swish", "residual", "relu"))}
    return {"op": op, "m": _log_int(rng, 1, 4096), "n": _log_int(rng, 64, 4096), "k": _log_int(rng, 64, 4096),
            "dtype": rng.choice(("f32", "bf16", "f16")), "epilogue": rng.choice(("none", "swish", "residual", "relu"))}


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
    """Rows of a residual stream: a few channels are much larger than the rest."""
    x = _normal(g, (rows, d))
    big = _randint(g, 0, d, (max(1, d // 128),), torch.int64)
    x[:, big] *= 8.0
    return x.to(TYPES[dtype])


def _cache(g, case, pages, filled):
    """k, v [pages][heads][page][dim] and, for codes, their scales."""
    heads = case.get("kv_heads", case["heads"])
    shape = (pages, heads, case["page"], case["dim"])
    kind = case["cache"]
    got = {}
    for name in ("k", "v"):
        if not filled:
            got[name] = torch.zeros(shape, device="cuda:0", dtype=TYPES[kind])
        elif kind == "int8":
            got[name] = _randint(g, -127, 128, shape, torch.int8)
        elif kind == "e4m3":
            got[name] = (_normal(g, shape, 120.0)).clamp_(-448.0, 448.0).to(TYPES[kind])
        else:
            got[name] = _normal(g, shape).to(TYPES[kind])
        if kind in TOP:
            top = torch.rand(shape[:3], generator=g, device="cuda:0") * 3.0 + 1.0
            got[name + "_scale"] = (top / TOP[kind]) if filled else torch.zeros(shape[:3], device="cuda:0")
    return got


def _slots(g, n, pages, page):
    """Distinct slots of n tokens, whole pages one after another, 1 row in 32 padding."""
    order = torch.randperm(pages, generator=g, device="cuda:0")
    s = (order[:, None] * page + torch.arange(page, device="cuda:0")).reshape(-1)[:n]
    pad = torch.rand((n,), generator=g, device="cuda:0") < 1.0 / 32
    return torch.where(pad, -1, s).to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    s = {"case": dict(case), "kept": {}}
    op = case["op"]
    if op in ("write", "read"):
        n, heads, dim, page = case["n"], case["heads"], case["dim"], case["page"]
        pages = (n + page - 1) // page + 3
        s["pages"] = pages
        # one page behind the cache's last: where the plain form puts padding rows
        s.update(_cache(g, case, pages + 1, op == "read"))
        s["slots"] = _slots(g, n, pages, page)
        if op == "write":
            for name in ("new_k", "new_v"):
                s[name] = _activations(g, n, heads * dim, case["dtype"])
        s["out_k"] = torch.zeros((n, heads * dim), device="cuda:0", dtype=TYPES[case["dtype"]])
        s["out_v"] = torch.zeros_like(s["out_k"])
    elif op == "attn":
        b, page, most = case["batch"], case["page"], case["len"]
        per = (most + page - 1) // page
        lens = torch.full((b,), most, device="cuda:0", dtype=torch.int32)
        if case["ragged"]:
            lens = _randint(g, 0, most + 1, (b,), torch.int32)
            lens[:1] = most
            lens[1:2] = 0
            lens[2:3] = 1
        s["lens"] = lens
        s["pages"] = b * per + 1
        table = torch.randperm(b * per, generator=g, device="cuda:0").reshape(b, per).to(torch.int32)
        used = torch.arange(per, device="cuda:0") * page < lens[:, None]
        s["table"] = torch.where(used, table, -1).to(torch.int32).contiguous()
        s.update(_cache(g, case, s["pages"], True))
        s["q"] = _normal(g, (b, case["heads"], case["dim"])).to(TYPES[case["dtype"]])
        s["out"] = torch.empty_like(s["q"])
        s["scale"] = 1.0 / math.sqrt(case["dim"])
    elif op == "norm":
        rows, d = case["rows"], case["d"]
        s["x"] = _activations(g, rows, d, case["dtype"])
        s["res"] = _activations(g, rows, d, case["dtype"])
        s["gamma"] = _normal(g, (d,), 0.1, 1.0)
        s["sum"], s["out"] = torch.empty_like(s["x"]), torch.empty_like(s["x"])
    else:
        m, n, k = case["m"], case["n"], case["k"]
        ld = (k + 15) // 16 * 16
        if op == "proj":
            s["x"] = _activations(g, m, k, case["dtype"])
            s["res"] = _activations(g, m, k, case["dtype"])
            s["gamma"] = _normal(g, (k,), 0.1, 1.0)
            s["sum"] = torch.empty_like(s["x"])
            s["codes"] = torch.zeros((m, ld), device="cuda:0", dtype=torch.int8)
            s["code_scale"] = torch.zeros((m,), device="cuda:0")
        else:
            s["codes"] = torch.zeros((m, ld), device="cuda:0", dtype=torch.int8)
            s["codes"][:, :k] = _normal(g, (m, k), 32.0).round_().clamp_(-127, 127).to(torch.int8)
            s["code_scale"] = torch.rand((m,), generator=g, device="cuda:0") * 0.03 + 0.01
        s["w"] = _randint(g, -127, 128, (k, n), torch.int8)
        s["w_scale"] = (torch.rand((n,), generator=g, device="cuda:0") + 0.5) * (0.02 / math.sqrt(k))
        s["bias"] = _normal(g, (n,), 0.1)
        s["stream"] = _activations(g, m, n, case["dtype"]) if case["epilogue"] == "residual" else None
        s["out"] = torch.empty((m, n), device="cuda:0", dtype=TYPES[case["dtype"]])
    return s


# ---- the plain forms ---------------------------------------------------------

def _quantised(x, top):
    """Codes (as fp32 whole numbers or unrounded e4m3 values) and scales of the last axis's rows."""
    amax = x.abs().amax(-1)
    zero = amax < TINY
    inv = torch.where(zero, 0.0, top / amax)
    return (x * inv[..., None]).clamp(-top, top), torch.where(zero, 0.0, amax / top)


def _plain_write(s):
    case = s["case"]
    n, heads, dim, page = case["n"], case["heads"], case["dim"], case["page"]
    slot = torch.where(s["slots"] < 0, s["pages"] * page, s["slots"]).long()
    at, off = slot // page, slot % page
    for name in ("k", "v"):
        x = s["new_" + name].float().reshape(n, heads, dim)
        if case["cache"] in TOP:
            codes, scale = _quantised(x, TOP[case["cache"]])
            if case["cache"] == "int8":
                codes = codes.round()
            s[name + "_scale"][at, :, off] = scale
            x = codes
        if case["cache"] == "e4m3":     # indexed stores go by bytes
            s[name].view(torch.uint8)[at, :, off] = x.to(TYPES["e4m3"]).view(torch.uint8)
        else:
            s[name][at, :, off] = x.to(TYPES[case["cache"]])
    return _plain_read(s)


def _plain_rows(s, name, at, off):
    got = s[name]
    if s["case"]["cache"] == "e4m3":
        got = got.view(torch.uint8)[at, :, off].view(TYPES["e4m3"])
    else:
        got = got[at, :, off]
    got = got.float()
    return got * s[name + "_scale"][at, :, off][..., None] if name + "_scale" in s else got


def _plain_read(s):
    case = s["case"]
    n, page = case["n"], case["page"]
    slot = s["slots"].long().clamp_min(0)
    there = (s["slots"] >= 0)[:, None, None]
    return [torch.where(there, _plain_rows(s, name, slot // page, slot % page), 0.0).reshape(n, -1)
            .to(TYPES[case["dtype"]]) for name in ("k", "v")]


def _plain_seen(s):
    """Positions of the longest sequence that each sequence's token sees."""
    case = s["case"]
    t = torch.arange(s["table"].shape[1] * case["page"], device="cuda:0")
    lens = s["lens"].long()[:, None]
    seen = t < lens
    return seen & (t >= lens - case["window"]) if case["window"] else seen


def _plain_attn(s):
    case = s["case"]
    b, heads, dim, kv = case["batch"], case["heads"], case["dim"], case["kv_heads"]
    table = s["table"].long().clamp_min(0)
    kind = case["cache"]

    def side(name):
        got = s[name].view(torch.uint8)[table].view(TYPES[kind]) if kind == "e4m3" else s[name][table]
        got = got.float()
        if kind in TOP:
            got = got * s[name + "_scale"][table][..., None]
        return got.transpose(1, 2).reshape(b * kv, -1, dim)        # [b kv][tokens][dim]

    q = s["q"].float().reshape(b * kv, heads // kv, dim).transpose(1, 2).contiguous()
    score = torch.matmul(side("k"), q) * s["scale"]                 # [b kv][tokens][group]
    seen = _plain_seen(s).repeat_interleave(kv, 0)[..., None]
    score = torch.where(seen, score, -torch.inf)
    top = score.amax(1, keepdim=True)
    p = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    total = p.sum(1, keepdim=True)
    p = (p / torch.where(total == 0.0, 1.0, total)).transpose(1, 2).contiguous()
    return torch.matmul(p, side("v")).reshape(b, heads, dim).to(s["q"].dtype)


def _plain_normed(s):
    """The stored sum and the fp32 norm of it."""
    h = (s["x"].float() + s["res"].float()).to(s["x"].dtype)
    eps = torch.tensor(EPS, dtype=torch.float32).item()
    mean = h.double().square().mean(-1, keepdim=True)       # 64 bits: codes lie next to borders
    r = (1.0 / torch.sqrt(mean + eps)).float()
    return h, (h.float() * r) * s["gamma"]


def _plain_gemm(s, codes, code_scale):
    case = s["case"]
    acc = torch.matmul(codes.float(), s["w"].float())
    y = acc * (code_scale[:, None] * s["w_scale"]) + s["bias"]
    if case["epilogue"] == "swish":
        y = y * (1.0 / (1.0 + torch.exp(-y)))
    elif case["epilogue"] == "relu":
        y = torch.where(y > 0.0, y, 0.0)
    elif case["epilogue"] == "residual":
        y = s["stream"].float() + y
    return y.to(TYPES[case["dtype"]])


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "write":
        return _plain_write(s)
    if op == "read":
        return _plain_read(s)
    if op == "attn":
        return _plain_attn(s)
    if op == "norm":
        h, y = _plain_normed(s)
        return h, y.to(s["x"].dtype)
    if op == "proj":
        h, y = _plain_normed(s)
        codes, scale = _quantised(y, TOP["int8"])
        return h, _plain_gemm(s, codes.round(), scale)
    return _plain_gemm(s, s["codes"][:, :case["k"]], s["code_scale"])


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
    return {"f32": pk.F32, "f16": pk.F16, "bf16": pk.BF16, "int8": pk.I8, "e4m3": pk.E4M3}[name]


def _own_cache(pk, s):
    """The cache's description: made once, as a program that holds the cache does."""
    kept = s["kept"]
    if "cache" not in kept:
        case = s["case"]
        scales = [s[n].data_ptr() if n in s else None for n in ("k_scale", "v_scale")]
        kept["cache"] = pk.KvCache(s["k"].data_ptr(), s["v"].data_ptr(), *scales, _kind(pk, case["cache"]),
                                   s["pages"], case["page"], case.get("kv_heads", case["heads"]), case["dim"])
        kept["cache_p"] = ctypes.byref(kept["cache"])
    return kept["cache_p"]


def _own_read(pk, s, stream):
    case = s["case"]
    wide = case["heads"] * case["dim"]
    pk.call("pk_gpu_kv_read_dev", _own_cache(pk, s), _kind(pk, case["dtype"]), s["slots"].data_ptr(), case["n"],
            s["out_k"].data_ptr(), wide, s["out_v"].data_ptr(), wide, stream)
    return [s["out_k"], s["out_v"]]


def _own_write(pk, s, stream):
    case = s["case"]
    wide = case["heads"] * case["dim"]
    pk.call("pk_gpu_kv_write_dev", _own_cache(pk, s), _kind(pk, case["dtype"]), s["new_k"].data_ptr(), wide,
            s["new_v"].data_ptr(), wide, s["slots"].data_ptr(), case["n"], stream)
    return _own_read(pk, s, stream)


def _own_attn(pk, s, stream):
    case, kept = s["case"], s["kept"]
    cache = _own_cache(pk, s)
    wide = case["heads"] * case["dim"]
    if "floats" not in kept:
        kept["floats"] = pk.load().pk_gpu_paged_attention_ws_floats(cache, case["batch"], case["heads"], case["len"],
                                                                    case["window"])
        kept["ws"] = torch.empty((max(1, kept["floats"]),), device="cuda:0")
    pk.call("pk_gpu_paged_attention_dev", cache, _kind(pk, case["dtype"]), s["q"].data_ptr(), wide, case["heads"],
            s["table"].data_ptr(), s["table"].shape[1], s["lens"].data_ptr(), case["batch"], case["len"],
            s["scale"], case["window"], s["out"].data_ptr(), wide, None, kept["ws"].data_ptr(), kept["floats"], stream)
    return s["out"]


def _own_gemm(pk, s, stream):
    case, kept = s["case"], s["kept"]
    m, n, k = case["m"], case["n"], case["k"]
    if "panel" not in kept:       # the weight in the kernels' order: made once, as a program does at load time
        kept["panel"] = torch.empty((pk.load().pk_gpu_w8_panel_bytes(k, n),), device="cuda:0", dtype=torch.uint8)
        pk.call("pk_gpu_w8_panel_dev", k, n, s["w"].data_ptr(), n, kept["panel"].data_ptr(), stream)
    epi = {"none": pk.EPI_NONE, "swish": pk.EPI_SWISH, "relu": pk.EPI_RELU, "residual": pk.EPI_RESIDUAL}[case["epilogue"]]
    res = s["stream"]
    pk.call("pk_gpu_gemm_w8a8_dev", m, n, k, s["codes"].data_ptr(), s["codes"].shape[1], s["code_scale"].data_ptr(),
            kept["panel"].data_ptr(), 1.0, s["w_scale"].data_ptr(), s["bias"].data_ptr(), epi,
            res.data_ptr() if res is not None else None, n, _kind(pk, case["dtype"]), s["out"].data_ptr(), n, stream)
    return s["out"]


def _own_norm(pk, s, stream, codes):
    x = s["x"]
    rows, d = x.shape
    kind = _kind(pk, s["case"]["dtype"])
    out, scale = (s["codes"], s["code_scale"].data_ptr()) if codes else (s["out"], None)
    pk.call("pk_gpu_rms_norm_dev", kind, x.data_ptr(), d, s["res"].data_ptr(), d, s["sum"].data_ptr(), d,
            s["gamma"].data_ptr(), EPS, pk.I8 if codes else kind, out.data_ptr(), out.shape[1], scale, rows, d, stream)
    return s["sum"], out


def _own(s):
    pk = _pk()
    stream = torch.cuda.current_stream().cuda_stream
    op = s["case"]["op"]
    if op == "write":
        return _own_write(pk, s, stream)
    if op == "read":
        return _own_read(pk, s, stream)
    if op == "attn":
        return _own_attn(pk, s, stream)
    if op == "norm":
        return _own_norm(pk, s, stream, False)
    if op == "proj":
        total, _ = _own_norm(pk, s, stream, True)
        return total, _own_gemm(pk, s, stream)
    return _own_gemm(pk, s, stream)


def run(state):
    return _own(state) if own else _plain(state)


# ---- work and exact values ---------------------------------------------------

def _tokens(case):
    """Tokens that the case's sequences attend over: those of ragged batches on average."""
    most, w = case["len"], case["window"]
    if not case["ragged"]:
        return case["batch"] * (min(most, w) if w else most)
    mean = most / 2 if not w else (w * (most - w) + w * w / 2) / most if w < most else most / 2
    return case["batch"] * mean


def work(case):
    op, size = case["op"], SIZE.get(case["dtype"], 4)
    if op in ("write", "read"):
        rows = 2 * case["n"] * case["heads"]
        held = rows * (case["dim"] * SIZE[case["cache"]] + (4 if case["cache"] in TOP else 0))
        given = rows * case["dim"] * size
        times = 2 if op == "write" else 1      # written, and read back
        return {"bytes": times * (held + given) + 4 * times * case["n"], "flops": 0}
    if op == "attn":
        t = _tokens(case)
        row = case["dim"] * SIZE[case["cache"]] + (4 if case["cache"] in TOP else 0)
        return {"bytes": 2 * t * case["kv_heads"] * row + 2 * case["batch"] * case["heads"] * case["dim"] * size,
                "flops": 4 * t * case["heads"] * case["dim"]}
    if op == "norm":
        n = case["rows"] * case["d"]
        return {"bytes": 4 * n * size + 4 * case["d"], "flops": 5 * n}
    m, n, k = case["m"], case["n"], case["k"]
    moved = m * k + k * n + m * n * size * (2 if case["epilogue"] == "residual" else 1) + 4 * (m + 2 * n)
    if op == "proj":      # rows, residual and sum, then the codes out and in again
        moved += m * k * (3 * size + 1) + 4 * k + 4 * m
    return {"bytes": moved, "flops": 2 * m * n * k}


def _nearest(x, top, kind):
    """In 64 bits: what the codes of the last axis's rows stand for."""
    big = x.abs().max(-1, keepdim=True).values
    unit = big / top
    y = torch.where(big < TINY, torch.zeros_like(x), x / unit.clamp_min(1e-300))
    if kind == "int8":
        return y.round() * unit
    # e4m3: 3 bits behind the leading one, exponents from -6 up
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp_min(2.0 ** -6))) - 3.0)
    return torch.round(y / step) * step * unit


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    kind = case.get("cache")
    if op == "write":
        keep = (s["slots"] >= 0).double()[:, None]
        got = []
        for x in (s["new_k"], s["new_v"]):
            x = x.double().view(case["n"], case["heads"], case["dim"])
            x = _nearest(x, TOP[kind], kind) if kind in TOP else x.to(TYPES[kind]).double()
            got.append(x.view(case["n"], -1) * keep)
        return got
    if op == "read":
        rows = s["slots"].long().clamp_min(0)
        got = []
        for name in ("k", "v"):
            flat = s[name].double().permute(0, 2, 1, 3).reshape(-1, case["heads"], case["dim"])
            x = flat.index_select(0, rows)
            if kind in TOP:
                x = x * s[name + "_scale"].double().permute(0, 2, 1).reshape(-1, case["heads"], 1).index_select(0, rows)
            got.append((x * (s["slots"] >= 0).double()[:, None, None]).reshape(case["n"], -1))
        return got
    if op == "attn":
        group = case["heads"] // case["kv_heads"]
        out = torch.zeros((case["batch"], case["heads"], case["dim"]), device="cuda:0", dtype=torch.float64)
        for b, n in enumerate(s["lens"].tolist()):
            first = max(0, n - case["window"]) if case["window"] else 0
            if n == first:
                continue
            pages = s["table"][b, first // case["page"]:(n - 1) // case["page"] + 1].long()
            at = first - first // case["page"] * case["page"]

            def side(name):
                x = s[name].view(torch.uint8)[pages].view(TYPES[kind]) if kind == "e4m3" else s[name][pages]
                x = x.double()
                if kind in TOP:
                    x = x * s[name + "_scale"][pages].double().unsqueeze(-1)
                return x.permute(1, 0, 2, 3).reshape(case["kv_heads"], -1, case["dim"])[:, at:at + n - first]

            q = s["q"][b].double().view(case["kv_heads"], group, case["dim"])
            w = torch.softmax(q @ side("k").transpose(1, 2).contiguous() / math.sqrt(case["dim"]), -1)
            out[b] = (w @ side("v")).reshape(case["heads"], case["dim"])
        return out
    if op in ("norm", "proj"):
        total = s["x"].double() + s["res"].double()
        held = total.to(torch.float32).to(s["x"].dtype).double()     # the norm is of the stored sum
        rms = torch.linalg.vector_norm(held, dim=-1, keepdim=True) / math.sqrt(held.shape[-1])
        y = held / torch.sqrt(rms * rms + EPS) * s["gamma"].double()
        if op == "norm":
            return total, y
        a = _nearest(y, 127.0, "int8")
    else:
        a = s["codes"][:, :case["k"]].double() * s["code_scale"].double().unsqueeze(1)
    z = a @ (s["w"].double() * s["w_scale"].double()) + s["bias"].double()
    if case["epilogue"] == "swish":
        z = z * torch.sigmoid(z)
    elif case["epilogue"] == "relu":
        z = z.clamp_min(0.0)
    elif case["epilogue"] == "residual":
        z = z + s["stream"].double()
    return (total, z) if op == "proj" else z
