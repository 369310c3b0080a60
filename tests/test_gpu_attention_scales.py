"""Attention where the scales of the cache's pages are far apart: zero, the smallest that are stored, and large ones in pages that
a query does not see.

The bound of an output is paged_ref.attention's: it is made of the values that the query sees, whatever the others are.
"""
import numpy as np
import pytest

import paged_ref as R
import test_gpu_attention as A

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f16", "bf16"]
# (lengths, new tokens, kv heads, group): one token, drafts, chunks of few columns, and prompts past them
SHAPES = {"step": ([200, 40, 90], [1, 1, 1], 2, 4), "draft": ([200, 70], [5, 3], 1, 4), "chunk": ([150, 96], [100, 60], 1, 3),
          "prompt": ([290], [263], 1, 8)}


def check(torch, c, window=0, **kw):
    """As test_gpu_attention.check, with nothing allowed beside the bound but the spacing of the type's smallest numbers."""
    got = A.run(torch, c, window, **kw)
    want, bound = R.attention(c["q"].float().numpy(), *c["codes"], *c["scale"], c["q_start"], c["lens"], c["table"],
                              c["hd"] ** -0.5, window, A.UNIT[c["dtype"]])
    far = np.abs(got - want)
    if c["dtype"] == "f16":  # (from 65520 on a result rounds to infinity: one that may lie there by its bound may be infinite)
        far[((got == np.inf) & (want + bound >= 65520)) | ((got == -np.inf) & (want - bound <= -65520))] = 0
    least = {"f32": 2.0 ** -145, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}[c["dtype"]]
    assert np.all(far <= bound + least), (float(np.nanmax(far / (bound + least))), bool(np.isnan(got).any()))


def first_pages(c, n, value, what=1):
    """The first n pages of every request (all: n = -1) at a scale of `value`."""
    for row in c["table"]:
        pages = row[row >= 0]
        c["scale"][what][pages if n < 0 else pages[:n]] = value


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("page,n", [(64, 1), (16, 2), (32, 1), (16, 5), (64, -1)])
def test_value_pages_of_zeros(gpu, dtype, shape, page, n):
    """Warm-up, padding, a value head that is zero: alone, and with other pages behind them."""
    lens, new, kv, grp = SHAPES[shape]
    c = A.case(gpu, dtype, lens, new, page, kv, grp, 64, seed=page + n)
    first_pages(c, n, 0.0)
    check(gpu, c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("page,n", [(64, 1), (16, 4), (16, 3), (64, -1)])
@pytest.mark.parametrize("largest", [2.0 ** -119, 2.0 ** -118, 2.0 ** -110])
def test_the_smallest_values_that_are_stored(gpu, dtype, shape, page, n, largest):
    """Pages whose largest value is just above what counts as zero: alone, and with ordinary pages behind them."""
    lens, new, kv, grp = SHAPES[shape]
    c = A.case(gpu, dtype, lens, new, page, kv, grp, 64, seed=page - n)
    first_pages(c, n, np.float32(largest) / np.float32(127))
    check(gpu, c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("ratio", [1e3, 1e6, 1e9])
@pytest.mark.parametrize("new,grp", [(100, 3), (270, 8)])
@pytest.mark.parametrize("held", [0, 5])
def test_later_pages_of_large_values(gpu, dtype, page, ratio, new, grp, held):
    """A prompt from its first token, and one behind a few: what a query does not see yet takes nothing from its result."""
    c = A.case(gpu, dtype, [held + new], [new], page, 1, grp, 64, seed=page)
    c["scale"][1][c["table"][0, 1]] *= ratio
    c["scale"][1][c["table"][0, 3 if page == 16 else 0]] *= 1 if page == 64 else 30
    check(gpu, c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("lens,new,grp,window", [([200, 130, 60], [1, 1, 1], 4, 9), ([200, 130], [20, 3], 4, 20), ([290], [263], 8, 17)])
def test_pages_before_the_window(gpu, dtype, page, lens, new, grp, window):
    """Large values that have left the window, beside small ones in it."""
    c = A.case(gpu, dtype, lens, new, page, 1, grp, 64, seed=page + window)
    for r, n in enumerate(lens):
        c["scale"][1][c["table"][r, :(n - new[r] - window) // page]] *= 1e8
        c["scale"][1][c["table"][r, 2]] *= 1e7
    check(gpu, c, window=window)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", list(SHAPES))
@pytest.mark.parametrize("page", [16, 64])
def test_missing_pages_beside_a_first_page_never_written(gpu, dtype, shape, page):
    """Table entries that are no pages, in a cache whose page 0 holds whatever was there before: NaN scales."""
    lens, new, kv, grp = SHAPES[shape]
    for seed in range(100):
        c = A.case(gpu, dtype, lens, new, page, kv, grp, 64, seed=seed, spare=6)
        if not (c["table"] == 0).any():
            break
    assert np.isnan(c["scale"][0][0]).all() and np.isnan(c["scale"][1][0]).all()
    c["table"][0, 1], c["table"][-1, 0] = -1, 2 ** 31 - 1
    check(gpu, c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("lens,new,grp,window", [([200, 130, 60], [1, 1, 1], 4, 9), ([200, 130], [20, 3], 4, 20), ([390], [263], 8, 17)])
def test_pages_that_no_query_sees_may_hold_anything(gpu, dtype, page, lens, new, grp, window):
    """Pages that a sliding window has left behind for good, never written since."""
    c = A.case(gpu, dtype, lens, new, page, 1, grp, 64, seed=page + window)
    for r, n in enumerate(lens):
        left = c["table"][r, :(n - new[r] - window + 1) // page]
        c["scale"][0][left] = c["scale"][1][left] = np.nan
    check(gpu, c, window=window)
