"""GPU: RMS norm of rows longer than registers hold, and of more rows than
workgroups in the kernels of 256 and 1024 threads a row.  Form and tolerances are
test_gpu_rms_norm's."""
import numpy as np
import pytest

import decode_oracle as do
from pkgpu import pk
from test_gpu_rms_norm import plain, test_against_plain_form as against_plain_form

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


@pytest.mark.parametrize("rows,D,kind,out,extra,off", [
    # the sum is stored and read again
    (3, 20001, "bf16", "int8", 0, 0), (2, 16385, "f32", "bf16", 3, 1), (2, 33000, "f16", "f16", 0, 3),
    (1030, 16390, "bf16", "int8", 0, 0),
    # a workgroup's second and third row
    (2500, 2304, "bf16", "int8", 0, 0), (2100, 2049, "f32", "int8", 0, 1), (1500, 4097, "f16", "int8", 0, 0),
    (2060, 8200, "bf16", "int8", 0, 0), (1100, 16384, "f16", "bf16", 0, 0),
])
def test_long_and_many(rows, D, kind, out, extra, off):
    against_plain_form(rows, D, kind, out, True, True, True, extra, off)


@pytest.mark.parametrize("over", ["x", "res"])
def test_long_rows_in_place(over):
    """The output over x or over the residual, with and without a stored sum over the other."""
    import torch
    rows, D = 3, 17001
    rng = np.random.default_rng(D)
    x, res = (rng.normal(0, 1, (rows, D)).astype(np.float32) for _ in range(2))
    h, y, _ = plain(x, res, None, 1e-6, "f32")
    for with_sum in (False, True):
        d = {"x": torch.from_numpy(x).to("cuda:0"), "res": torch.from_numpy(res).to("cuda:0")}
        other = d["res" if over == "x" else "x"]
        pk.call("pk_gpu_rms_norm_dev", pk.F32, d["x"].data_ptr(), D, d["res"].data_ptr(), D,
                other.data_ptr() if with_sum else None, D, None, 1e-6, pk.F32, d[over].data_ptr(), D, None, rows, D,
                do.stream())
        torch.cuda.synchronize()
        assert np.array_equal(do.values(d[over]), y.astype(np.float64))
        assert np.array_equal(do.values(other), (h if with_sum else res if over == "x" else x).astype(np.float64))


def test_the_longest_row():
    """2^31 - 1 elements, a pattern of 4096 over and over: indices past 2^31 - 1024 stay in the row.

    The fp64 sum is off by 2^21 additions of a thread's, 2^-32; r, h * r and the output's rounding are the others."""
    import torch
    D = (1 << 31) - 1
    base = torch.from_numpy(np.random.default_rng(1).normal(0, 1, 4096).astype(np.float32)).to(torch.bfloat16)
    x = torch.empty((D + 1,), dtype=torch.bfloat16, device="cuda:0")
    x.view(-1, 4096).copy_(base.to("cuda:0"))
    out = torch.full((D + 1,), 5.0, dtype=torch.bfloat16, device="cuda:0")
    pk.call("pk_gpu_rms_norm_dev", pk.BF16, x.data_ptr(), D, None, 0, None, 0, None, 1e-5, pk.BF16, out.data_ptr(), D,
            None, 1, D, do.stream())
    torch.cuda.synchronize()
    assert float(out[D]) == 5.0
    b = do.values(base)
    mean = ((b ** 2).sum() * (1 << 19) - b[-1] ** 2) / D
    want = b / np.sqrt(mean + np.float64(np.float32(1e-5)))
    out[D] = out[4095]
    got = out.view(-1, 4096)
    assert bool((got == got[0]).all())
    assert np.all(np.abs(do.values(got[0]) - want) <= np.abs(want) * (3.01 * 2.0 ** -24 + 2.0 ** -31 + 2.0 ** -8 * 1.01))
