"""GPU: the kernel of many rows by two sides (two waves with the same rows, half of each tile's
tokens each) with infinities and NaN in the tokens of one side, and with the narrowest window."""
import numpy as np
import pytest
import torch

import more_oracle as mo
from pkgpu import pk
from prompt_call import prompt, sides
from test_gpu_prompt_attention_many import TWO

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", autouse=True)
def ready():
    pk.call("pk_gpu_init", 0)


NEW, LENS = [70, 0, 33, 129], [470, 40, 450, 431]


def places(c, b, t):
    return int(c.table_h[b, t // 16]), t % 16


def put(c, at, bad):
    """`bad` into element 5 of the first head's value and 6 of the others'; codes: a NaN for all of the token."""
    page, off = at
    if c.cache.kind in ("int8", "e4m3"):
        c.cache.part("v_scale")[page, :, off] = float("nan")
    elif c.cache.kind == "e2m1":
        c.cache.part("v_scale")[page, :, off, :] = 255
    else:
        v = c.cache.part("v")
        v[page, 0, off, 5] = bad
        v[page, 1:, off, 6] = bad


def expect(c, want, got, rows, bad):
    """Rows `rows` carry it, everything else is as without it."""
    got = got.copy()
    if c.cache.kind in ("int8", "e4m3", "e2m1"):
        assert np.isnan(got[rows]).all()
        got[rows] = want.out[rows]
    else:
        g = c.heads // c.cache.heads
        for part in (np.s_[:g, 5], np.s_[g:, 6]):
            x = got[rows][(slice(None),) + part]
            assert np.array_equal(x, np.full(x.shape, bad), equal_nan=True)
            got[(rows,) + part] = want.out[(rows,) + part]
    live = want.live >= 0
    tol = want.bound(c.cache.kind, c.rows, mo.half_of_weights(c.cache.kind, c.rows, True))
    assert np.all((np.abs(got - want.out) <= tol)[live])


@pytest.mark.parametrize("kind,rows,dim", TWO)
@pytest.mark.parametrize("token", [
    366,          # new, in the second half of a tile: side 1's, which the last 65 rows see
    334,          # new, in the first half
    40, 10,       # behind all of the sequence's rows
])
def test_what_is_not_finite_in_one_side(kind, rows, dim, token):
    rng = np.random.default_rng(dim + len(kind))
    c = prompt(rng, kind, rows, 11, 3, dim, 16, NEW, LENS, tail=5, pad=64)
    assert c.many() and sides(c) == 2
    want = c.plain()
    pos = np.arange(c.n) - c.starts_h[3] + LENS[3] - NEW[3]
    carry = np.flatnonzero((want.live == 3) & (pos >= token))
    assert len(carry) == (129 if token < 302 else 431 - token)
    for bad in (float("inf"), -float("inf"), float("nan")):
        put(c, places(c, 3, token), bad)
        expect(c, want, c.run(want), carry, float("nan") if kind in ("int8", "e4m3", "e2m1") else bad)


@pytest.mark.parametrize("kind,rows,dim", TWO)
def test_keys_that_are_not_finite(kind, rows, dim):
    """A NaN of a key makes its head's rows NaN that see it, and no others; the lse too."""
    rng = np.random.default_rng(dim)
    c = prompt(rng, kind, rows, 11, 3, dim, 16, NEW, LENS, tail=5)
    assert c.many() and sides(c) == 2
    want = c.plain()
    pos = np.arange(c.n) - c.starts_h[3] + LENS[3] - NEW[3]
    for token in (366, 334):
        page, off = places(c, 3, token)
        if kind in ("int8", "e4m3"):
            c.cache.part("k_scale")[page, 2, off] = float("nan")
        elif kind == "e2m1":
            c.cache.part("k_scale")[page, 2, off, 1] = 255
        else:
            c.cache.part("k")[page, 2, off, 9] = float("nan")
        got = c.run(want)
        carry = np.flatnonzero((want.live == 3) & (pos >= token))
        lse = c.lse[:c.n].cpu().numpy()
        assert np.isnan(got[carry][:, 6:9]).all() and np.isnan(lse[carry][:, 6:9]).all()
        got[carry[:, None], np.arange(6, 9)] = want.out[carry[:, None], np.arange(6, 9)]
        live = want.live >= 0
        tol = want.bound(kind, rows, mo.half_of_weights(kind, rows, True))
        assert np.all((np.abs(got - want.out) <= tol)[live])


@pytest.mark.parametrize("kind,dim", [("bf16", 64), ("bf16", 128), ("int8", 64), ("int8", 128), ("e4m3", 128), ("e2m1", 128),
                                      ("f16", 64)])
def test_values_near_the_largest_float(kind, dim):
    """Sums of one side, or of both, that leave their range: the rows again, one by one."""
    rng = np.random.default_rng(dim)
    rows = "f16" if kind == "f16" else "bf16"
    c = prompt(rng, kind, rows, 11, 3, dim, 16, NEW, LENS, tail=5)
    assert c.many() and sides(c) == 2
    if kind == "f16":                                     # its largest values stay within f32: no row is taken again
        c.cache.part("v")[c.table_h[2, 6]] = 65504.0
        c.check()
        return
    for tokens in (slice(0, 8), slice(8, 16)):            # pages of 16: tokens 96 to 111, side 1's, then also 64 to 79
        page = c.table_h[2, 6 if tokens.start == 0 else 4]
        if kind == "bf16":
            c.cache.part("v")[page, :, tokens] = 3e38
        elif kind == "e2m1":
            c.cache.part("v_scale")[page, :, tokens] = 252
        else:
            c.cache.part("v_scale")[page, :, tokens] = 1e36 if kind == "int8" else 5e35
        c.check(more=2.0 ** -18)


@pytest.mark.parametrize("kind,rows,dim", TWO)
@pytest.mark.parametrize("window", [1, 2, 33])
def test_narrow_windows(kind, rows, dim, window):
    """Rows that see themselves alone: of every tile of tokens most waves' halves hold nothing."""
    rng = np.random.default_rng(dim + window)
    c = prompt(rng, kind, rows, 33, 2, dim, 16, [360], [459], window=window)
    assert c.many() and sides(c) == 2
    c.check()


def test_a_document_of_one_token_each():
    """The same by `first`, and rows whose range is empty between them."""
    rng = np.random.default_rng(2)
    for kind, rows in (("bf16", "bf16"), ("int8", "f16"), ("e2m1", "f32")):
        c = prompt(rng, kind, rows, 33, 2, 128, 16, [360], [459], first=lambda b, p: np.where(p % 5 == 0, 1 << 30, p))
        assert c.many() and sides(c) == 2
        got, want = c.check(), c.plain()
        assert (want.seen == 0).sum() == 72 and np.all(got[want.seen == 0] == 0)
        assert bool(torch.isneginf(c.lse[:c.n][torch.from_numpy(want.seen == 0).to("cuda:0")]).all())
