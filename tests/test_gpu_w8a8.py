"""GPU: int8 rows x int8 weights with an epilogue, against whole sums in 64 bits.

Tolerance: the sum to fp32, the scales' product, their product and the bias are
four roundings of at most 2^-24 each of |v| or |v - bias|, the residual one
more, Swish 2^-21 of its value (16-bit outputs: and 2^-24 |v| of it) and its slope (at most 1.1) times v's error, the
output half a step of its type."""
import numpy as np
import pytest

import decode_oracle as do
from pkgpu import pk

pytestmark = pytest.mark.gpu

EPI = {"none": pk.EPI_NONE, "swish": pk.EPI_SWISH, "half": pk.EPI_HALF_RESIDUAL, "residual": pk.EPI_RESIDUAL,
       "relu": pk.EPI_RELU}


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


def panel_of(w, ldb=None):
    import torch
    K, N = w.shape
    ldb = ldb or N
    t = torch.full((K, ldb), 99, dtype=torch.int8, device="cuda:0")
    t[:, :N] = torch.from_numpy(w).to("cuda:0")
    n = pk.load().pk_gpu_w8_panel_bytes(K, N)
    p = torch.full((n + 64,), 0x5A, dtype=torch.uint8, device="cuda:0")
    pk.call("pk_gpu_w8_panel_dev", K, N, t.data_ptr(), ldb, p.data_ptr(), do.stream())
    torch.cuda.synchronize()
    assert bool((p[n:] == 0x5A).all())
    return p


def plain(a, sa, w, sb, bias, epi, res):
    """Outputs in 64 bits and their fp32 operations' error bound."""
    acc = np.rint(a.astype(np.float64) @ w.astype(np.float64))      # whole: below 2^53
    s = acc * sa[:, None].astype(np.float64) * np.asarray(sb, np.float64)
    v = s + (0 if bias is None else bias.astype(np.float64))
    e = 2.0 ** -24 * (3.01 * np.abs(s) + 1.01 * np.abs(v))
    if epi == "swish":
        y = v / (1 + np.exp(-v))
        return y, 1.1 * e + (2.0 ** -21 + 2.0 ** -24 * np.abs(v)) * np.abs(y)
    if epi == "relu":
        return np.maximum(v, 0), e
    if epi in ("half", "residual"):
        y = res.astype(np.float64) + (0.5 if epi == "half" else 1.0) * v
        return y, e + 2.0 ** -24 * 1.01 * np.abs(y)
    return v, e


CASES = [
    # M, N, K, type, epilogue, extra lda, extra ldc, scales per column, bias
    (1, 16, 16, "f32", "none", 0, 0, True, True), (1, 1, 1, "f32", "none", 0, 0, False, False),
    (1, 1000, 1024, "bf16", "swish", 0, 0, True, True), (16, 130, 65, "f16", "relu", 16, 1, True, True),
    (17, 64, 4096, "f32", "residual", 0, 0, False, True), (33, 4096, 1024, "f32", "swish", 0, 0, True, True),
    (48, 257, 1000, "bf16", "half", 0, 7, True, False), (64, 31, 300, "f32", "none", 32, 1, True, True),
    (65, 129, 127, "f32", "residual", 0, 3, True, True), (100, 96, 128, "f16", "swish", 0, 0, False, True),
    (300, 260, 129, "bf16", "relu", 0, 0, True, True), (1111, 1023, 777, "bf16", "residual", 0, 1, True, True),
    (2000, 2304, 256, "f32", "swish", 0, 0, True, True), (4001, 4096, 384, "bf16", "swish", 0, 0, True, True),
    (3500, 4100, 1024, "f16", "half", 0, 0, True, True),
    (3200, 1024, 1100, "f32", "relu", 0, 0, True, True), (3200, 1024, 100, "bf16", "none", 0, 0, True, True),
    (2000, 2500, 650, "bf16", "half", 16, 0, True, True), (4001, 4001, 130, "f16", "none", 0, 0, True, True),
    (130, 300, 700, "f32", "residual", 0, 1, True, True), (250, 100, 64, "bf16", "swish", 0, 0, True, True),
    (40, 2100, 333, "f16", "relu", 0, 0, True, True), (50, 4200, 260, "f32", "half", 0, 0, True, True),
    (70, 65, 513, "f32", "none", 0, 0, True, True), (200, 500, 2049, "f32", "swish", 0, 0, True, True),
]


def run(M, N, K, kind, epi, xa, xc, per_col, with_bias, a, sa, w, sb, bias, res, in_place=False):
    import torch
    lda, ldc = (K + 15) // 16 * 16 + xa, N + xc
    da = torch.full((M, lda), -77, dtype=torch.int8, device="cuda:0")      # past K: anything
    da[:, :K] = torch.from_numpy(a).to("cuda:0")
    tt = do.torch_type(kind)
    out = torch.full((M * ldc + 64,), 5.0, dtype=tt, device="cuda:0")
    C = out[:M * ldc].view(M, ldc)
    dres = None
    if res is not None:
        dres = C if in_place else torch.full((M, ldc), 3.0, dtype=tt, device="cuda:0")
        dres[:, :N] = torch.from_numpy(res).to(tt).to("cuda:0")
    dsa = torch.from_numpy(sa).to("cuda:0")
    dsb = torch.from_numpy(sb).to("cuda:0") if per_col else None
    db = torch.from_numpy(bias).to("cuda:0") if with_bias else None
    p = panel_of(w, N + (5 if N % 2 else 0))
    ptr = lambda t: t.data_ptr() if t is not None else None
    pk.call("pk_gpu_gemm_w8a8_dev", M, N, K, da.data_ptr(), lda, dsa.data_ptr(), p.data_ptr(),
            float(sb) if not per_col else 123.0, ptr(dsb), ptr(db), EPI[epi], ptr(dres), ldc, do.FLOATS[kind],
            C.data_ptr(), ldc, do.stream())
    torch.cuda.synchronize()
    got = do.values(C)
    assert np.all(got[:, N:] == 5) and bool((out[M * ldc:] == 5).all())
    return got[:, :N]


@pytest.mark.parametrize("M,N,K,kind,epi,xa,xc,per_col,with_bias", CASES)
def test_against_plain_form(M, N, K, kind, epi, xa, xc, per_col, with_bias):
    rng = np.random.default_rng(M + N + K)
    a = rng.integers(-128, 128, (M, K)).astype(np.int8)
    w = rng.integers(-128, 128, (K, N)).astype(np.int8)
    sa = rng.uniform(0.5, 2, M).astype(np.float32) / 127
    sb = (rng.uniform(0.5, 2, N) / (60 * np.sqrt(K))).astype(np.float32) if per_col else np.float32(0.001)
    bias = rng.normal(0, 0.5, N).astype(np.float32) if with_bias else None
    res = do.rounded(rng.normal(0, 1, (M, N)), kind) if epi in ("half", "residual") else None
    want, e = plain(a, sa, w, sb, bias, epi, res)
    tol = e + do.HALF[kind] * 1.01 * (np.abs(want) + e) + 2.0 ** -25
    for in_place in ((False, True) if res is not None else (False,)):
        got = run(M, N, K, kind, epi, xa, xc, per_col, with_bias, a, sa, w, sb, bias, res, in_place)
        err = np.abs(got - want)
        assert np.all(err <= tol), (float((err - tol).max()), np.argwhere(err > tol)[:4].tolist())


@pytest.mark.parametrize("M", [3, 130])
def test_the_largest_sums(M):
    """K = 131071 of the most negative codes: 2^31 - 16384, the largest sum there is."""
    import torch
    K, N = 131071, 24
    lda = 131072
    a = torch.full((M, lda), -128, dtype=torch.int8, device="cuda:0")
    w = np.full((K, N), -128, np.int8)
    w[:, 1] = 127
    p = panel_of(w)
    one = torch.ones((M,), device="cuda:0")
    C = torch.zeros((M, N), device="cuda:0")
    pk.call("pk_gpu_gemm_w8a8_dev", M, N, K, a.data_ptr(), lda, one.data_ptr(), p.data_ptr(), 1.0, None, None,
            pk.EPI_NONE, None, 0, pk.F32, C.data_ptr(), N, do.stream())
    torch.cuda.synchronize()
    want = np.full((M, N), np.float32(128 * 128 * 131071), np.float64)
    want[:, 1] = np.float32(-128 * 127 * 131071)
    assert np.array_equal(do.values(C), want)


def test_rows_without_a_finite_scale_stay_theirs():
    """A row whose scale is NaN is NaN; its neighbours are not touched by it."""
    rng = np.random.default_rng(0)
    M, N, K = 70, 40, 100
    a = rng.integers(-127, 128, (M, K)).astype(np.int8)
    w = rng.integers(-127, 128, (K, N)).astype(np.int8)
    sa = np.full(M, 0.01, np.float32)
    sa[9] = np.nan
    sb = np.full(N, 0.01, np.float32)
    got = run(M, N, K, "f32", "swish", 0, 0, True, False, a, sa, w, sb, None, None)
    assert np.isnan(got[9]).all() and np.isfinite(np.delete(got, 9, 0)).all()


def test_swish_far_out():
    """-110 to 110 and beyond, by way of the bias.  exp2 and the reciprocal are off by 2^-23 each, four
    roundings by 2^-24 each at most: 2^-21.  Where the reciprocal of e^-v leaves the normal range
    (v < -87.3) -0 stands for up to 87.4 / 2^126 < 2^-119."""
    import torch
    N = 4096
    v = np.concatenate([np.linspace(-110, 110, N - 6), [-3e38, 3e38, -88.5, -87.3, 0.0, -0.0]]).astype(np.float32)
    p = panel_of(np.zeros((16, N), np.int8))
    a = torch.zeros((1, 16), dtype=torch.int8, device="cuda:0")
    one, b = torch.ones((1,), device="cuda:0"), torch.from_numpy(v).to("cuda:0")
    C = torch.zeros((1, N), device="cuda:0")
    pk.call("pk_gpu_gemm_w8a8_dev", 1, N, 16, a.data_ptr(), 16, one.data_ptr(), p.data_ptr(), 1.0, None, b.data_ptr(),
            pk.EPI_SWISH, None, 0, pk.F32, C.data_ptr(), N, do.stream())
    torch.cuda.synchronize()
    x = v.astype(np.float64)
    with np.errstate(over="ignore"):
        want = x / (1 + np.exp(-x))
    assert np.all(np.abs(do.values(C)[0] - want) <= 2.0 ** -21 * np.abs(want) + 2.0 ** -119)


def test_a_norm_feeds_a_product():
    """RMS norm's codes through the product, replayed from a graph with new rows."""
    import torch
    rng = np.random.default_rng(5)
    for M in (5, 200):
        K, N = 320, 192
        w = rng.integers(-127, 128, (K, N)).astype(np.int8)
        p = panel_of(w)
        sb = (rng.uniform(0.5, 1.5, N) / 2000).astype(np.float32)
        dsb = torch.from_numpy(sb).to("cuda:0")
        x = torch.zeros((M, K), device="cuda:0")
        codes = torch.zeros((M, K), dtype=torch.int8, device="cuda:0")
        sc = torch.zeros((M,), device="cuda:0")
        C = torch.zeros((M, N), device="cuda:0")
        g, s = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=s):
            pk.call("pk_gpu_rms_norm_dev", pk.F32, x.data_ptr(), K, None, 0, None, 0, None, 1e-5, pk.I8,
                    codes.data_ptr(), K, sc.data_ptr(), M, K, s.cuda_stream)
            pk.call("pk_gpu_gemm_w8a8_dev", M, N, K, codes.data_ptr(), K, sc.data_ptr(), p.data_ptr(), 1.0,
                    dsb.data_ptr(), None, pk.EPI_RELU, None, 0, pk.F32, C.data_ptr(), N, s.cuda_stream)
        for _ in range(3):
            xs = rng.normal(0, 1, (M, K)).astype(np.float32)
            x.copy_(torch.from_numpy(xs))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            want, e = plain(codes.cpu().numpy(), sc.cpu().numpy(), w, sb, None, "relu", None)
            assert np.all(np.abs(do.values(C) - want) <= e + 2.0 ** -23 * np.abs(want))
            # and the whole is what fp32 rows give, to the codes' half steps
            y = xs.astype(np.float64) / np.sqrt((xs.astype(np.float64) ** 2).mean(-1, keepdims=True) + 1e-5)
            half = 0.51 * np.abs(y).max(-1, keepdims=True) / 127
            far = half * np.abs(w.astype(np.float64)).sum(0) * sb
            assert np.all(np.abs(do.values(C) - np.maximum(y @ (w * sb.astype(np.float64)), 0)) <= far)


def test_empty_sizes():
    for M, N in ((0, 8), (8, 0)):
        pk.call("pk_gpu_gemm_w8a8_dev", M, N, 16, None, 16, None, None, 1.0, None, None, pk.EPI_NONE, None, 0, pk.F32,
                None, 8, do.stream())
