"""CPU: what the decoder operators refuse, before any device is touched.

Pointers here are small aligned numbers that nothing may dereference."""
import ctypes

import pytest

from pkgpu import gpu_available, pk

P = 1 << 20             # an aligned address no call may read


def cache(**kw):
    d = dict(k=P, v=P, k_scale=P, v_scale=P, dtype=pk.I8, n_pages=4, page_size=16, heads=2, head_dim=128)
    d.update(kw)
    return pk.KvCache(*[d[n] for n, _ in pk.KvCache._fields_])


def refused(fn, *args, code=-1, text=None):
    lib = pk.load()
    assert getattr(lib, fn)(*args) == code
    msg = lib.pk_gpu_last_error().decode()
    assert msg and (text is None or text in msg), msg


def attention(code=-1, text=None, **kw):
    d = dict(c=None, dtype=pk.F32, q=P, ldq=512, heads=4, pages=P, ld_pages=8, lens=P, B=3, max_len=128, scale=1.0,
             window=0, out=P, ldo=512, lse=None, ws=P, floats=1 << 30)
    d.update(kw)
    refused("pk_gpu_paged_attention_dev", *d.values(), None, code=code, text=text)


BAD_CACHES = [
    (dict(k=None), -1, "NULL"), (dict(v=None), -1, "NULL"), (dict(k_scale=None), -1, "NULL"),
    (dict(v_scale=None), -1, "NULL"), (dict(k=P + 8), -1, "aligned"), (dict(v_scale=P + 4), -1, "aligned"),
    (dict(dtype=pk.F32), -1, "type"), (dict(dtype=9), -1, "type"), (dict(head_dim=96), -2, "head_dim"),
    (dict(head_dim=0), -2, "head_dim"), (dict(page_size=8), -2, "page_size"), (dict(page_size=48), -2, "page_size"),
    (dict(page_size=0), -2, "page_size"), (dict(page_size=-16), -2, "page_size"), (dict(n_pages=0), -1, "pages"),
    (dict(heads=0), -1, "heads"), (dict(n_pages=1 << 28), -1, "2^31"), (dict(heads=1 << 25), -1, "2^31"),
]


@pytest.mark.parametrize("bad,code,text", BAD_CACHES)
def test_bad_caches(bad, code, text):
    c = ctypes.byref(cache(**bad))
    refused("pk_gpu_kv_write_dev", c, pk.F32, P, 1 << 30, P, 1 << 30, P, 1, None, code=code, text=text)
    refused("pk_gpu_kv_read_dev", c, pk.F32, P, 1, P, 1 << 30, P, 1 << 30, None, code=code, text=text)
    attention(c=c, ldq=1 << 30, ldo=1 << 30, heads=1 << 25 if bad.get("heads") else 2, code=code, text=text)
    assert pk.load().pk_gpu_paged_attention_ws_floats(c, 1, 2, 1000, 0) == 0


def test_16_bit_caches_need_no_scales():
    c = cache(dtype=pk.BF16, k_scale=None, v_scale=None)
    refused("pk_gpu_kv_write_dev", ctypes.byref(c), pk.F32, None, 256, P, 256, P, 1, None, text="NULL operand")


@pytest.mark.parametrize("dtype,k,ldk,v,ldv,slots,n,text", [
    (pk.I8, P, 256, P, 256, P, 1, "type"), (-1, P, 256, P, 256, P, 1, "type"),
    (pk.F32, P, 255, P, 256, P, 1, "ldk"), (pk.F32, P, 256, P, 0, P, 1, "ldv"),
    (pk.F32, P, 256, P, 256, P, -1, "n ="), (pk.F32, None, 256, P, 256, P, 1, "NULL"),
    (pk.F32, P, 256, None, 256, P, 1, "NULL"), (pk.F32, P, 256, P, 256, None, 1, "NULL"),
    (pk.F32, P + 4, 256, P, 256, P, 1, "aligned"), (pk.BF16, P, 256, P, 260, P, 1, "aligned"),
    (pk.F32, P, 256, P, 256, P, 1 << 30, "2^31"), (pk.F32, P, 256, P, 256, P + 2, 1, "aligned"),
])
def test_bad_rows(dtype, k, ldk, v, ldv, slots, n, text):
    c = ctypes.byref(cache())
    refused("pk_gpu_kv_write_dev", c, dtype, k, ldk, v, ldv, slots, n, None, text=text)
    refused("pk_gpu_kv_read_dev", c, dtype, slots, n, k, ldk, v, ldv, None, text=text)


def test_null_cache():
    refused("pk_gpu_kv_write_dev", None, pk.F32, P, 256, P, 256, P, 1, None, text="NULL cache")
    refused("pk_gpu_kv_read_dev", None, pk.F32, P, 1, P, 256, P, 256, None, text="NULL cache")


@pytest.mark.parametrize("kw,code,text", [
    (dict(dtype=pk.I8), -1, "type"), (dict(dtype=7), -1, "type"), (dict(heads=0), -1, "heads"),
    (dict(heads=3), -1, "heads"), (dict(heads=-2), -1, "heads"), (dict(B=-1), -1, "B ="),
    (dict(max_len=-1), -1, "max_len"), (dict(max_len=(1 << 30) + 1), -1, "max_len"), (dict(window=-1), -1, "window"),
    (dict(ldq=511), -1, "ldq"), (dict(ldo=511), -1, "ldo"), (dict(ld_pages=7), -1, "pages"),
    (dict(ld_pages=-1), -1, "pages"), (dict(q=None), -1, "NULL"), (dict(out=None), -1, "NULL"),
    (dict(lens=None), -1, "NULL"), (dict(pages=None), -1, "NULL"), (dict(q=P + 8), -1, "aligned"),
    (dict(out=P + 4), -1, "aligned"), (dict(ldq=513), -1, "aligned"), (dict(ldo=514), -1, "aligned"),
    (dict(B=1 << 30), -1, "grid"), (dict(pages=P + 1), -1, "aligned"), (dict(lens=P + 2), -1, "aligned"),
    (dict(lse=P + 3), -1, "aligned"),
])
def test_bad_attention(kw, code, text):
    attention(c=ctypes.byref(cache()), code=code, text=text, **kw)


@pytest.mark.parametrize("held,dtype", [(pk.F16, pk.F32), (pk.F16, pk.BF16), (pk.BF16, pk.F16)])
def test_queries_a_16_bit_cache_does_not_take(held, dtype):
    attention(c=ctypes.byref(cache(dtype=held)), dtype=dtype, code=-2, text="queries")


def test_attention_workspace():
    c = ctypes.byref(cache())
    lib = pk.load()
    need = lib.pk_gpu_paged_attention_ws_floats(c, 3, 4, 1000, 0)
    assert need > 0 and need % (3 * 4 * 130) == 0
    for ws, floats in ((None, need), (P, need - 1), (P + 4, need)):
        attention(c=c, max_len=1000, ld_pages=63, ws=ws, floats=floats, text="workspace")
    assert lib.pk_gpu_paged_attention_ws_floats(c, 3, 4, 32, 0) == 0         # one chunk
    assert lib.pk_gpu_paged_attention_ws_floats(c, 0, 4, 1000, 0) == 0
    assert lib.pk_gpu_paged_attention_ws_floats(c, 3, 3, 1000, 0) == 0       # refused sizes
    assert lib.pk_gpu_paged_attention_ws_floats(c, 3, 4, 1000, 64) <= need   # a window needs no more


def norm(code=-1, text=None, **kw):
    d = dict(dtype=pk.F32, x=P, ldx=64, res=P + 4096, ldr=64, sum=P + 8192, lds=64, gamma=P, eps=1e-5, out_dtype=pk.I8,
             out=P + 12288, ldo=64, scales=P, rows=2, D=64)
    d.update(kw)
    refused("pk_gpu_rms_norm_dev", *d.values(), None, code=code, text=text)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=pk.I8), "type"), (dict(dtype=-1), "type"), (dict(out_dtype=pk.E4M3), "type"),
    (dict(out_dtype=12), "type"), (dict(rows=-1), "rows"), (dict(D=0), "D ="), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(ldx=63), "leading"), (dict(ldr=63), "leading"), (dict(lds=63), "leading"),
    (dict(ldo=63), "leading"), (dict(x=None), "NULL"), (dict(out=None), "NULL"), (dict(scales=None), "NULL"),
    (dict(x=P + 2), "aligned"), (dict(res=P + 1), "aligned"), (dict(sum=P + 3), "aligned"),
    (dict(out=P + 2, out_dtype=pk.F32), "aligned"), (dict(gamma=P + 2), "aligned"), (dict(scales=P + 1), "aligned"),
    (dict(out=P), "in place"), (dict(out=P, out_dtype=pk.F32, ldo=72), "in place"),
    (dict(out=P + 4096, out_dtype=pk.F16), "in place"), (dict(sum=P, lds=65), "in place"),
    (dict(sum=P + 4096, lds=72), "in place"), (dict(sum=P + 12288), "in place"),
])
def test_bad_norms(kw, text):
    norm(text=text, **kw)


def gemm(code=-1, text=None, **kw):
    d = dict(M=4, N=32, K=64, A=P, lda=64, sa=P, panel=P, B_scale=1.0, sb=P, bias=P, epi=pk.EPI_RESIDUAL, res=P, ldr=32,
             dtype=pk.BF16, C=P, ldc=32)
    d.update(kw)
    refused("pk_gpu_gemm_w8a8_dev", *d.values(), None, code=code, text=text)


@pytest.mark.parametrize("kw,text", [
    (dict(M=-1), "M ="), (dict(N=-1), "N ="), (dict(N=(1 << 30) + 1, ldc=(1 << 30) + 1), "N ="), (dict(K=0), "K ="),
    (dict(K=131072, lda=131072), "K ="), (dict(dtype=pk.I8), "type"), (dict(epi=5), "epilogue"),
    (dict(epi=-1), "epilogue"), (dict(lda=72), "lda"), (dict(lda=48), "lda"),
    (dict(lda=(1 << 27) + 16), "lda"), (dict(M=(1 << 30) + 1), "M ="), (dict(ldc=31), "ldc"),
    (dict(ldr=31), "ldr"), (dict(A=None), "NULL"), (dict(sa=None), "NULL"), (dict(panel=None), "NULL"),
    (dict(C=None), "NULL"), (dict(res=None), "NULL"), (dict(A=P + 8), "aligned"), (dict(panel=P + 8), "aligned"),
    (dict(C=P + 1), "aligned"), (dict(res=P + 1), "aligned"), (dict(sa=P + 2), "aligned"), (dict(sb=P + 2), "aligned"),
    (dict(bias=P + 1), "aligned"), (dict(ldr=40), "in place"),
])
def test_bad_products(kw, text):
    gemm(text=text, **kw)


def test_bad_panels():
    lib = pk.load()
    assert lib.pk_gpu_w8_panel_bytes(1, 1) == 2048 and lib.pk_gpu_w8_panel_bytes(129, 17) == 2 * 2 * 2048
    for K, N in ((0, 1), (1, 0), (-1, 5), (131072, 1), (1, (1 << 30) + 1)):
        assert lib.pk_gpu_w8_panel_bytes(K, N) == 0
        refused("pk_gpu_w8_panel_dev", K, N, P, max(N, 1), P, None)
    refused("pk_gpu_w8_panel_dev", 16, 16, P, 15, P, None, text="ldb")
    refused("pk_gpu_w8_panel_dev", 16, 16, None, 16, P, None, text="NULL")
    refused("pk_gpu_w8_panel_dev", 16, 16, P, 16, None, None, text="NULL")
    refused("pk_gpu_w8_panel_dev", 16, 16, P, 16, P + 8, None, text="aligned")


@pytest.mark.skipif(gpu_available(), reason="checks the no-device error path")
def test_no_device_is_an_error_for_every_operator():
    """Good arguments without a device: PK_GPU_ENODEV, with rows and without any."""
    c = ctypes.byref(cache())
    for n in (1, 0):
        refused("pk_gpu_kv_write_dev", c, pk.F32, P, 256, P, 256, P, n, None, code=-5)
        refused("pk_gpu_kv_read_dev", c, pk.F32, P, n, P, 256, P, 256, None, code=-5)
        attention(c=c, B=n, code=-5)
        norm(rows=n, code=-5)
        gemm(M=n, code=-5)
    refused("pk_gpu_w8_panel_dev", 16, 16, P, 16, P, None, code=-5)
