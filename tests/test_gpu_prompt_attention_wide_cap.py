"""Attention with rules, caps far above the scores.  GPU: f32 queries keep units of the score as long as
scale / cap is a normal float.  CPU: below that the call is refused."""
import numpy as np
import pytest

from pkgpu import gpu_available, pk
from prompt_call import prompt
from test_prompt_refusals import attention, rules


@pytest.mark.gpu
@pytest.mark.parametrize("scale,cap", [(0.9e-6, 1e30), (-0.9e-6, 7e31), (0.9e-6, 2.0 ** 105)])
@pytest.mark.parametrize("new,kv", [(4, 2), (140, 64)])
def test_caps_far_above_the_scores(scale, cap, new, kv):
    pk.call("pk_gpu_init", 0)
    rng = np.random.default_rng(new)
    c = prompt(rng, "bf16", "f32", kv, 2, 64, 16, [new], [150], scale=scale, cap=cap)
    assert c.many() == (new > 4)
    c.q_h *= 2.0 ** 20                                    # scores of some units
    c.q *= 2.0 ** 20
    c.check()


BELOW = [(0.9e-6, 1e36), (2.0 ** -7, 2.0 ** 120), (1e-38, 1.0), (-1e-6, 1e36), (1e-45, 1e-3)]


@pytest.mark.parametrize("scale,cap", BELOW)
@pytest.mark.parametrize("dtype", [pk.F32, pk.BF16])
def test_quotients_below_a_normal_float_are_refused(scale, cap, dtype):
    attention(rules=rules(scale=scale, cap=cap), dtype=dtype, text="cap")


@pytest.mark.skipif(gpu_available(), reason="makes calls with addresses that nothing may read")
@pytest.mark.parametrize("scale,cap", [(0.0, 50.0), (2.0 ** -6, 2.0 ** 120), (-(2.0 ** -6), 2.0 ** 120), (2.0 ** -126, 1.0), (1e-45, 0.0)])
def test_quotients_that_are_not(scale, cap):
    attention(rules=rules(scale=scale, cap=cap), code=-5)
