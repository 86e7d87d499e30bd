"""GPU: one decoder block's step as a program runs it, captured once and
replayed token by token: norm of the residual stream to codes, the fused QKV
product, the cache write, attention over the cache, the output projection on
the framework's own int8 GEMM, a second norm, the feed-forward's up product
with Swish and its down projection into the stream.

Every stage of every replay is checked against its 64-bit form on the stage's
own inputs as the device holds them, within that operator's bound."""
import numpy as np
import pytest

import decode_oracle as do
from pkgpu import pk
from test_gpu_rms_norm import plain as plain_norm
from test_gpu_w8a8 import panel_of, plain as plain_gemm

pytestmark = pytest.mark.gpu

B, H, KV, DIM, D, FF, PAGE, STEPS = 5, 4, 2, 64, 256, 320, 16, 35
QKV = (H + 2 * KV) * DIM
EPS = 1e-5


class Block:
    def __init__(self, kind):
        import torch
        rng = np.random.default_rng(3)
        per = (STEPS + PAGE - 1) // PAGE
        self.cache = do.Cache(kind, B * per, KV, PAGE, DIM, filled=False)
        self.st = self.cache.struct()
        self.table_h = rng.permutation(B * per).reshape(B, per).astype(np.int32)
        z = lambda *s, dtype=torch.float32: torch.zeros(s, dtype=dtype, device="cuda:0")
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")
        self.table = put(self.table_h)
        self.lens, self.slots = z(B, dtype=torch.int32), z(B, dtype=torch.int32)
        self.x, self.add, self.stream = z(B, D), z(B, D), z(B, D)
        self.codes, self.sc = z(B, D, dtype=torch.int8), z(B)
        self.codes2, self.sc2 = z(B, D, dtype=torch.int8), z(B)
        self.qkv, self.att, self.up = z(B, QKV), z(B, H * DIM), z(B, FF)
        self.mid, self.out = z(B, D), z(B, D)
        self.w = {n: rng.integers(-127, 128, s).astype(np.int8)
                  for n, s in (("qkv", (D, QKV)), ("o", (H * DIM, D)), ("up", (D, FF)), ("down", (FF, D)))}
        self.ws = {n: (rng.uniform(0.5, 1.5, w.shape[1]) / (60 * np.sqrt(w.shape[0]))).astype(np.float32)
                   for n, w in self.w.items()}
        self.g = {n: rng.normal(1, 0.1, D).astype(np.float32) for n in ("n1", "n2")}
        self.bias = rng.normal(0, 0.1, QKV).astype(np.float32)
        self.d = {n: put(v) for n, v in list(self.g.items()) + [("bias", self.bias), ("wo", self.w["o"]),
                                                                   ("wd", self.w["down"])]}
        self.dws = {n: put(v) for n, v in self.ws.items()}
        self.panels = {n: panel_of(self.w[n]) for n in ("qkv", "up")}
        self.floats = pk.load().pk_gpu_paged_attention_ws_floats(do.ref(self.st), B, H, STEPS, 0)
        self.work = z(self.floats + 4)

    def enqueue(self, s):
        p = lambda t: t.data_ptr()
        pk.call("pk_gpu_rms_norm_dev", pk.F32, p(self.x), D, p(self.add), D, p(self.stream), D, p(self.d["n1"]), EPS,
                pk.I8, p(self.codes), D, p(self.sc), B, D, s)
        pk.call("pk_gpu_gemm_w8a8_dev", B, QKV, D, p(self.codes), D, p(self.sc), p(self.panels["qkv"]), 0.0,
                p(self.dws["qkv"]), p(self.d["bias"]), pk.EPI_NONE, None, 0, pk.F32, p(self.qkv), QKV, s)
        k = p(self.qkv) + 4 * H * DIM
        pk.call("pk_gpu_kv_write_dev", do.ref(self.st), pk.F32, k, QKV, k + 4 * KV * DIM, QKV, p(self.slots), B, s)
        pk.call("pk_gpu_paged_attention_dev", do.ref(self.st), pk.F32, p(self.qkv), QKV, H, p(self.table),
                self.table.shape[1], p(self.lens), B, STEPS, 0.125, 0, p(self.att), H * DIM, None, p(self.work),
                self.floats, s)
        self.mid.copy_(self.stream)
        pk.call("pk_gpu_gemm_i8_ex_dev", B, D, H * DIM, 1.0, p(self.att), H * DIM, p(self.d["wo"]), 0.001, D, 0.0,
                p(self.mid), D, None, pk.EPI_RESIDUAL, s)
        pk.call("pk_gpu_rms_norm_dev", pk.F32, p(self.mid), D, None, 0, None, 0, p(self.d["n2"]), EPS, pk.I8,
                p(self.codes2), D, p(self.sc2), B, D, s)
        pk.call("pk_gpu_gemm_w8a8_dev", B, FF, D, p(self.codes2), D, p(self.sc2), p(self.panels["up"]), 0.0,
                p(self.dws["up"]), None, pk.EPI_SWISH, None, 0, pk.F32, p(self.up), FF, s)
        self.out.copy_(self.mid)
        pk.call("pk_gpu_gemm_i8_ex_dev", B, D, FF, 1.0, p(self.up), FF, p(self.d["wd"]), 0.001, D, 0.0,
                p(self.out), D, None, pk.EPI_RESIDUAL, s)

    def check_codes(self, x, gamma, codes, sc):
        _, y, _ = plain_norm(x, None, gamma, EPS, "f32")
        want, scale = do.codes(y, "int8")
        assert np.array_equal(do.values(codes), want.astype(np.float64))
        assert np.array_equal(do.values(sc), scale.astype(np.float64))

    def check(self, t, x, add):
        f32 = lambda t: t.detach().cpu().numpy()
        assert np.array_equal(f32(self.stream), x + add)
        self.check_codes(f32(self.stream), self.g["n1"], self.codes, self.sc)
        want, e = plain_gemm(f32(self.codes), f32(self.sc), self.w["qkv"], self.ws["qkv"], self.bias, "none", None)
        qkv = f32(self.qkv).astype(np.float64)
        assert np.all(np.abs(qkv - want) <= e + 2.0 ** -23 * np.abs(want))
        new = self.table_h[:, t // PAGE] * PAGE + t % PAGE
        for i, name in enumerate(("k", "v")):
            rows = qkv[:, (H + i * KV) * DIM:(H + (i + 1) * KV) * DIM].reshape(B, KV, DIM)
            assert np.all(np.abs(self.cache.rows(name)[new] - rows) <= do.code_bound(rows, self.cache.kind))
        q = qkv[:, :H * DIM].reshape(B, H, DIM)
        lens = [t + 1] * B
        want, _, a, s, xx = do.attention(self.cache, q, self.table_h, lens, STEPS, 0.125, 0)
        att = f32(self.att).astype(np.float64).reshape(B, H, DIM)
        assert np.all(np.abs(att - want) <= do.attention_bound(want, a, s, xx, t + 1, DIM, self.cache.kind, "f32"))
        # the framework's own GEMM: within 1e-3 of the largest value, as it states
        for src, w, res, got in ((att.reshape(B, -1), self.w["o"], self.stream, self.mid),
                                 (f32(self.up).astype(np.float64), self.w["down"], self.mid, self.out)):
            prod = src @ (w.astype(np.float64) * np.float64(np.float32(0.001)))
            err = np.abs(f32(got).astype(np.float64) - (f32(res).astype(np.float64) + prod))
            assert err.max() <= 1e-3 * np.abs(prod).max() + 2.0 ** -23 * np.abs(f32(got)).max()
        self.check_codes(f32(self.mid), self.g["n2"], self.codes2, self.sc2)
        want, e = plain_gemm(f32(self.codes2), f32(self.sc2), self.w["up"], self.ws["up"], None, "swish", None)
        assert np.all(np.abs(f32(self.up) - want) <= e + 2.0 ** -23 * np.abs(want))


@pytest.mark.parametrize("kind", ["int8", "e4m3", "bf16"])
def test_block_step_by_step(kind):
    import torch
    pk.call("pk_gpu_init", 0)
    b = Block(kind)
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        b.enqueue(s.cuda_stream)
    rng = np.random.default_rng(7)
    for t in range(STEPS):
        x, add = (rng.normal(0, 1, (B, D)).astype(np.float32) for _ in range(2))
        b.x.copy_(torch.from_numpy(x))
        b.add.copy_(torch.from_numpy(add))
        b.lens.fill_(t + 1)
        b.slots.copy_(torch.from_numpy((b.table_h[:, t // PAGE] * PAGE + t % PAGE).astype(np.int32)))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        b.check(t, x, add)
    assert b.cache.guards_whole()
