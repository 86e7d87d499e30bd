"""GPU: int8 products on both sides of each border between the kernels: 1, 2 or 3
blocks of rows a workgroup of the few-row kernel (the last of them not whole), and the tiles
that take over.  Form and tolerance are test_gpu_w8a8's."""
import numpy as np
import pytest

import decode_oracle as do
from pkgpu import pk
from test_gpu_w8a8 import plain, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [
    (16, 4096, 200), (17, 4095, 200), (17, 4097, 130), (32, 4080, 64), (33, 4080, 77), (33, 4096, 321), (48, 4081, 128),
    (48, 8192, 96), (48, 8193, 96), (49, 3008, 160), (64, 3008, 500), (64, 3009, 129), (100, 1472, 1000), (145, 960, 90),
    (700, 256, 64), (769, 256, 64), (3000, 60, 200), (3009, 60, 200),
])
def test_both_sides_of_each_border(M, N, K):
    pk.call("pk_gpu_init", 0)
    rng = np.random.default_rng(M * N + K)
    a = rng.integers(-128, 128, (M, K)).astype(np.int8)
    w = rng.integers(-128, 128, (K, N)).astype(np.int8)
    sa = rng.uniform(0.5, 2, M).astype(np.float32) / 127
    sb = (rng.uniform(0.5, 2, N) / (60 * np.sqrt(K))).astype(np.float32)
    bias = rng.normal(0, 0.5, N).astype(np.float32)
    want, e = plain(a, sa, w, sb, bias, "none", None)
    got = run(M, N, K, "f32", "none", 0, 0, True, True, a, sa, w, sb, bias, None)
    assert np.all(np.abs(got - want) <= e + do.HALF["f32"] * 1.01 * (np.abs(want) + e))
