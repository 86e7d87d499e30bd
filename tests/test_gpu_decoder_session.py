"""GPU: the operators of a decoder's sessions together, as a program runs them: prompts of several
sequences into the paged cache and attended at once, a second ragged chunk of each, single
tokens, drafted tokens, the last two captured once and replayed.

Rows come as a fused projection leaves them (queries, keys, values side by side), queries turn in
place.  Every stage of every replay is checked against its 64-bit form on the stage's own inputs
as the device holds them, within that operator's bound."""
import ctypes

import numpy as np
import pytest

import decode_oracle as do
import more_oracle as mo
from pkgpu import pk
from prompt_call import many_rows
from test_gpu_rope import freqs_of, kv_bound

pytestmark = pytest.mark.gpu

B, PAGE, LONGEST = 3, 16, 400


class Session:
    def __init__(self, kind, rows, heads, kv, dim, rot, interleaved, cap, bias, window):
        import torch
        self.kind, self.rows, self.heads, self.kv, self.dim, self.rot, self.inter = kind, rows, heads, kv, dim, rot, interleaved
        self.rng = np.random.default_rng(dim + heads)
        per = LONGEST // PAGE
        self.cache = mo.cache_of(kind, B * per, kv, PAGE, dim, seed=4)
        self.st = self.cache.struct()
        self.table_h = self.rng.permutation(B * per).reshape(B, per).astype(np.int32)
        put = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to("cuda:0")
        self.table = put(self.table_h)
        self.f = freqs_of(rot)
        self.d_f = put(self.f)
        self.rope = pk.Rope(self.d_f.data_ptr(), 1.0, rot, int(interleaved))
        slopes = (2.0 ** -np.arange(1, heads + 1)).astype(np.float32) if bias else None
        self.d_slopes = put(slopes) if bias else None
        self.how = dict(scale=dim ** -0.5, cap=cap, slopes=slopes, window=window)
        self.rules = pk.AttentionRules(dim ** -0.5, cap, self.d_slopes.data_ptr() if bias else None, window, None, None)
        self.lens_h = np.zeros(B, np.int32)

    def stage(self, most, max_new):
        return Stage(self, most, max_new)


class Stage:
    """Buffers of a call over up to `most` rows, max_new of a sequence, at addresses that stay."""

    def __init__(self, s, most, max_new):
        import torch
        self.s, self.most, self.max_new = s, most, max_new
        z = lambda *d, dtype=torch.int32: torch.zeros(d, dtype=dtype, device="cuda:0")
        tt = do.torch_type(s.rows)
        self.wide = (s.heads + 2 * s.kv) * s.dim
        self.qkv, self.out = z(most, self.wide, dtype=tt), z(most, s.heads * s.dim, dtype=tt)
        self.lse = z(most, s.heads, dtype=torch.float32)
        self.pos, self.slots, self.lens, self.starts = z(most), z(most), z(B), z(B + 1)
        self.floats = pk.load().pk_gpu_prompt_attention_ws_floats(do.ref(s.st), B, most, s.heads, max_new, LONGEST,
                                                                  s.how["window"])
        self.ws = z(self.floats + 4, dtype=torch.float32)

    def enqueue(self, stream):
        s, es = self.s, self.qkv.element_size()
        q = self.qkv.data_ptr()
        k = q + s.heads * s.dim * es
        pk.call("pk_gpu_rope_kv_write_dev", ctypes.byref(s.rope), do.ref(s.st), do.FLOATS[s.rows], q, self.wide, s.heads, q,
                self.wide, k, self.wide, k + s.kv * s.dim * es, self.wide, self.pos.data_ptr(), self.slots.data_ptr(),
                self.most, stream)
        pk.call("pk_gpu_prompt_attention_dev", do.ref(s.st), do.FLOATS[s.rows], q, self.wide, s.heads, s.table.data_ptr(),
                s.table.shape[1], self.lens.data_ptr(), self.starts.data_ptr(), B, self.most, self.max_new, LONGEST,
                ctypes.byref(s.rules), self.out.data_ptr(), s.heads * s.dim, self.lse.data_ptr(), self.ws.data_ptr(),
                self.floats, stream)

    def fill(self, new):
        """The next new[b] tokens of each sequence, padding behind them."""
        import torch
        s = self.s
        self.new = np.asarray(new)
        self.starts_h = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        n = int(self.starts_h[-1])
        self.b_of = np.repeat(np.arange(B), self.new)
        self.pos_h, self.slots_h = np.zeros(self.most, np.int32), np.full(self.most, -1, np.int32)
        self.pos_h[:n] = np.concatenate([s.lens_h[b] + np.arange(k) for b, k in enumerate(self.new)])
        self.slots_h[:n] = s.table_h[self.b_of, self.pos_h[:n] // PAGE] * PAGE + self.pos_h[:n] % PAGE
        s.lens_h = s.lens_h + self.new.astype(np.int32)
        self.qkv_h = do.rounded(s.rng.normal(0, 1, (self.most, self.wide)), s.rows)
        self.qkv.copy_(torch.from_numpy(self.qkv_h).to(self.qkv.dtype))
        for t, h in ((self.pos, self.pos_h), (self.slots, self.slots_h), (self.lens, s.lens_h), (self.starts, self.starts_h)):
            t.copy_(torch.from_numpy(h))
        self.out.fill_(7.0)
        self.lse.fill_(7.0)
        self.before = {m: s.cache.rows(m) for m in ("k", "v")}
        torch.cuda.synchronize()

    def check(self):
        import torch
        torch.cuda.synchronize()
        s, n = self.s, int(self.starts_h[-1])
        cut = lambda i, j, h: self.qkv_h[:, i * s.dim:j * s.dim].reshape(self.most, h, s.dim)
        q, k, v = cut(0, s.heads, s.heads), cut(s.heads, s.heads + s.kv, s.kv), cut(s.heads + s.kv, s.heads + 2 * s.kv, s.kv)
        # queries, turned in place
        got = do.values(self.qkv)
        want, size = mo.turned(q, self.pos_h, s.f, 1.0, s.rot, s.inter)
        held = got[:, :s.heads * s.dim].reshape(want.shape)
        assert np.all(np.abs(held - want) <= mo.turned_bound(want, size, s.rows, LONGEST))
        assert np.array_equal(got[:, s.heads * s.dim:], self.qkv_h[:, s.heads * s.dim:])
        # the cache: the new rows, and no other
        at = self.slots_h[:n]
        want, size = mo.turned(k[:n], self.pos_h[:n], s.f, 1.0, s.rot, s.inter)
        now = {m: s.cache.rows(m) for m in ("k", "v")}
        assert np.all(np.abs(now["k"][at] - want) <= kv_bound(want, size, s.kind, s.rows, LONGEST))
        val = v[:n].astype(np.float64)
        assert np.all(np.abs(now["v"][at] - val) <= kv_bound(val, np.zeros_like(val), s.kind, s.rows, 0.0))
        rest = np.ones(len(now["k"]), bool)
        rest[at] = False
        for m in ("k", "v"):
            assert np.array_equal(now[m][rest], self.before[m][rest])
        assert s.cache.guards_whole()
        # attention over both
        plain = mo.Ruled(s.cache, held, s.table_h, s.lens_h, self.starts_h, self.max_new, LONGEST,
                         exact_tanh=s.rows == "f32", **s.how)
        many = many_rows(s.kind, s.rows, s.kv, s.heads // s.kv, B, min(self.max_new, self.most), LONGEST, s.how["window"])
        tol = plain.bound(s.kind, s.rows, mo.half_of_weights(s.kind, s.rows, many))
        out = do.values(self.out).reshape(held.shape)
        err = np.abs(out - plain.out)[:n]
        assert np.all(err <= tol[:n]), (float((err / tol[:n]).max()), np.argwhere(err > tol[:n])[:4].tolist())
        assert np.all(np.abs(do.values(self.lse)[:n] - plain.lse[:n]) <= plain.lse_bound()[:n])
        assert np.all(out[n:] == 7) and bool((self.lse[n:] == 7).all())
        return many


@pytest.mark.parametrize("kind,rows,heads,kv,dim,rot,interleaved,cap,bias,window", [
    ("e2m1", "bf16", 8, 2, 128, 128, False, 0.0, False, 0), ("e2m1", "f32", 16, 16, 64, 32, True, 20.0, True, 0),
    ("int8", "bf16", 32, 32, 64, 64, False, 30.0, False, 100), ("bf16", "bf16", 24, 8, 256, 64, True, 0.0, True, 0),
    ("f16", "f16", 16, 16, 128, 128, False, 0.0, False, 90), ("e4m3", "f16", 12, 3, 128, 96, False, 50.0, True, 0),
])
def test_sessions(kind, rows, heads, kv, dim, rot, interleaved, cap, bias, window):
    import torch
    pk.call("pk_gpu_init", 0)
    s = Session(kind, rows, heads, kv, dim, rot, interleaved, cap, bias, window)
    for new, most in (([37, 150, 9], 200), ([110, 1, 64], 175)):         # prompts, then a chunk of each
        st = s.stage(most, max(new))
        st.fill(new)
        st.enqueue(do.stream())
        st.check()
    stream, graphs = torch.cuda.Stream(), []
    for st in (s.stage(B, 1), s.stage(5 * B, 5)):                         # a token each; up to five drafted
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=stream):
            st.enqueue(stream.cuda_stream)
        graphs.append((st, g))
    for i in range(3):
        for (st, g), new in zip(graphs, ([1, 1, 1], [[5, 3, 1], [1, 0, 4], [5, 5, 5]][i])):
            st.fill(new)
            g.replay()
            st.check()
    # a session's tokens taken back: what was drafted past them is not seen, and written over
    s.lens_h = s.lens_h - np.array([3, 0, 5], np.int32)
    graphs[0][0].fill([1, 1, 1])
    graphs[0][1].replay()
    graphs[0][0].check()
    # a sequence that has no new token this time
    graphs[0][0].fill([1, 0, 1])
    graphs[0][1].replay()
    graphs[0][0].check()


@pytest.mark.parametrize("kind", ["e2m1", "int8", "bf16"])
def test_one_token_is_the_one_token_attention(kind):
    """Over what a session wrote, a single token without rules is what pk_gpu_paged_attention_dev gives, within both
    bounds: once each."""
    import torch
    pk.call("pk_gpu_init", 0)
    s = Session(kind, "bf16", 8, 2, 128, 128, False, 0.0, False, 0)
    st = s.stage(200, 150)
    st.fill([37, 150, 9])
    st.enqueue(do.stream())
    st.check()
    one = s.stage(B, 1)
    one.fill([1, 1, 1])
    one.enqueue(do.stream())
    one.check()
    floats = pk.load().pk_gpu_paged_attention_ws_floats(do.ref(s.st), B, s.heads, LONGEST, 0)
    ws, out = torch.zeros(floats + 4, device="cuda:0"), torch.zeros_like(one.out)
    pk.call("pk_gpu_paged_attention_dev", do.ref(s.st), pk.BF16, one.qkv.data_ptr(), one.wide, s.heads, s.table.data_ptr(),
            s.table.shape[1], one.lens.data_ptr(), B, LONGEST, s.how["scale"], 0, out.data_ptr(), s.heads * s.dim, None,
            ws.data_ptr(), floats, do.stream())
    torch.cuda.synchronize()
    held = do.values(one.qkv)[:, :s.heads * s.dim].reshape(B, s.heads, s.dim)
    plain = mo.Ruled(s.cache, held, s.table_h, s.lens_h, np.arange(B + 1), 1, LONGEST, **s.how)
    tol = plain.bound(kind, "bf16", mo.half_of_weights(kind, "bf16", False))
    assert np.all(np.abs(do.values(out).reshape(held.shape) - plain.out) <= tol)
    assert np.all(np.abs(do.values(out) - do.values(one.out)).reshape(held.shape) <= 2 * tol)
