"""GPU: attention with rules, slopes up to the largest float: a token's own score stays, all others leave."""
import numpy as np
import pytest

from pkgpu import pk
from prompt_call import prompt

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


@pytest.mark.parametrize("kind,rows", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("int8", "bf16"), ("e2m1", "f32")])
@pytest.mark.parametrize("new,kv", [(4, 2), (140, 32)])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_slopes_near_the_largest_float(kind, rows, new, kv, cap):
    rng = np.random.default_rng(new)
    top = float(np.finfo(np.float32).max)
    slopes = np.tile(np.array([2.4e38, 3e38, top, 1e30], np.float32), kv // 2)
    c = prompt(rng, kind, rows, kv, 2, 64, 16, [new], [150], slopes=slopes, cap=cap)
    assert c.many() == (new > 4)
    got = c.check()
    v = c.cache.rows("v")                                  # each row is its own token's value
    # times its one weight over the sum of weights: over codes the weight carries the row's scale and is rounded, to
    # bf16 where rows are many (2^-8 of it), and so is the output (2^-8): (1 + 2^-8)^2 - 1 <= 2.01 * 2^-8
    off = 2.01 * 2.0 ** -8
    for r in range(c.n):
        t = 150 - new + r
        own = np.repeat(v[c.table_h[0, t // 16] * 16 + t % 16], 2, 0)
        assert np.all(np.abs(got[r] - own) <= off * np.abs(own))
