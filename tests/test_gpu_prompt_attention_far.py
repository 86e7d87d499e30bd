"""GPU: attention with rules over sequences that are split, where a token that a row sees weighs
nothing: an infinity or a NaN of its value is passed on all the same, as it is by a call that
takes the sequence whole, and what a row does not see stays out."""
import numpy as np
import pytest
import torch

import decode_oracle as do
import more_oracle as mo
from pkgpu import pk
from prompt_call import Prompt
from test_gpu_prompt_attention_many import splits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


DIM, KV, GROUP, PAGE = 64, 2, 2, 16


def two_calls(kind, rows, new, length, slope, first=None):
    """The same sequence in chunks and whole: with sequences of no new tokens behind it, and rows of no sequence,
    there are more tiles than the card has CUs, and none is split."""
    rng = np.random.default_rng(new)
    per = -(-length // PAGE)
    cache = mo.cache_of(kind, per + 1, KV, PAGE, DIM, seed=4)
    table = np.full((300, per), 1 << 30, np.int32)
    table[0] = rng.permutation(cache.pages)[:per]
    many = new > 8
    n = 8192 if many else new
    q = do.rounded(rng.normal(0, 1, (n, KV * GROUP, DIM)), rows).astype(np.float64)
    how = dict(slopes=np.full(KV * GROUP, slope, np.float32), first=None)
    calls = []
    for whole in (False, True):
        r = n if whole and many else new
        B = 300 if whole and not many else 1
        if first is not None:
            how["first"] = np.full(r, first, np.int32)
        starts = np.full(B + 1, new, np.int32)
        starts[0] = 0
        calls.append(Prompt(cache, q[:r], rows, table[:B], [length] + [0] * (B - 1), starts, new, length, DIM ** -0.5, **how))
        assert calls[-1].many() == many
    calls[1].floats = 0                                   # and it takes no workspace
    return calls


def values_at(calls, t):
    """Page and place of token t."""
    return int(calls[0].table_h[0, t // PAGE]), t % PAGE


def put(cache, at, kind, bad):
    """`bad` into a token's value of both heads; codes: a NaN scale, or byte."""
    page, off = at
    if kind in ("int8", "e4m3"):
        cache.part("v_scale")[page, :, off] = float("nan")
    elif kind == "e2m1":
        cache.part("v_scale")[page, :, off, :] = 255
    else:
        cache.part("v")[page, 0, off, 5], cache.part("v")[page, 1, off, 6] = bad, -bad


def outputs(calls, new):
    got = []
    for c in calls:
        c.out.fill_(5.0)
        c.lse.fill_(5.0)
        c.ws.fill_(float("nan"))
        assert c is calls[1] or splits(c) > 4
        c.enqueue(do.stream())
        torch.cuda.synchronize()
        assert bool((c.out[new:] == 5).all())
        got.append((do.values(c.out)[:new].reshape(new, KV * GROUP, DIM), do.values(c.lse)[:new]))
    return got


PAIRS = [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("int8", "bf16"), ("e4m3", "f32"), ("e2m1", "f16")]


CODES = ("int8", "e4m3", "e2m1")                          # are finite themselves: a NaN is their scale's


@pytest.mark.parametrize("kind,rows,bad", [(k, r, b) for k, r in PAIRS for b in (float("inf"), float("nan"))
                                           if k not in CODES or b != b])
@pytest.mark.parametrize("new,length", [(3, 4000), (300, 14000)])
@pytest.mark.parametrize("slope", [0.5, 1e38])
def test_a_seen_value_that_weighs_nothing(kind, rows, new, length, slope, bad):
    """Token 2, thousands of tokens back, behind a slope that leaves it no weight (1e38: not even a score)."""
    calls = two_calls(kind, rows, new, length, slope)
    want = calls[0].plain()                               # of the finite cache
    put(calls[0].cache, values_at(calls, 2), kind, bad)
    tol = want.bound(kind, rows, calls[0].half_p())
    for got, lse in outputs(calls, new):
        if kind in CODES:
            assert np.isnan(got).all()
            continue
        for h, e, x in ((0, 5, bad), (1, 5, bad), (2, 6, -bad), (3, 6, -bad)):
            assert np.array_equal(got[:, h, e], np.full(new, x), equal_nan=True), (h, got[:, h, e][:4])
            got[:, h, e] = want.out[:, h, e]
        assert np.all(np.abs(got - want.out) <= tol)
        assert np.all(np.abs(lse - want.lse) <= want.lse_bound())


@pytest.mark.parametrize("kind,rows", PAIRS)
@pytest.mark.parametrize("new,length", [(3, 4000), (300, 14000)])
def test_a_value_that_no_row_sees(kind, rows, new, length):
    """The same token before the first that rows see, in a chunk that holds nothing else of theirs."""
    calls = two_calls(kind, rows, new, length, 0.5, first=40)
    want = calls[0].plain()
    put(calls[0].cache, values_at(calls, 2), kind, float("nan"))
    tol = want.bound(kind, rows, calls[0].half_p())
    for got, lse in outputs(calls, new):
        assert np.all(np.abs(got - want.out) <= tol)
        assert np.all(np.abs(lse - want.lse) <= want.lse_bound())


@pytest.mark.parametrize("new,length", [(3, 4000), (300, 14000)])
def test_infinities_of_both_signs_and_a_key(new, length):
    """In different chunks, they make a NaN of the element; a NaN of a key one of the row."""
    calls = two_calls("bf16", "bf16", new, length, 0.5)
    v = calls[0].cache.part("v")
    for t, x in ((2, float("inf")), (length - new - 1, -float("inf"))):
        page, off = values_at(calls, t)
        v[page, 0, off, 5] = x
    for got, _ in outputs(calls, new):
        assert np.isnan(got[:, :2, 5]).all()
        got[:, :2, 5] = 0
        assert np.isfinite(got).all()
    page, off = values_at(calls, 2)
    calls[0].cache.part("k")[page, 1, off, 9] = float("nan")
    for got, lse in outputs(calls, new):
        assert np.isnan(got[:, 2:]).all() and np.isnan(lse[:, 2:]).all() and np.isfinite(lse[:, :2]).all()
