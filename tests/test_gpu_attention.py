"""Attention over the paged 8-bit cache on the GPU against a plain implementation in 64 bits.

The bound of each output is derived in paged_ref.attention from the roundings the kernels make.
"""
import numpy as np
import pytest

import jk
import paged_ref as R

pytestmark = pytest.mark.gpu

# roundings of the probabilities (f32: two f16 parts, 22 bits, and 2^-25 of the largest; else f16) and of the output
UNIT = {"f32": (2.0 ** -21, 2.0 ** -23), "f16": (2.0 ** -10, 2.0 ** -11), "bf16": (2.0 ** -10, 2.0 ** -8)}


def case(torch, dtype, lens, new, page, kv, grp, hd, seed=0, spare=3, outlier=True):
    rng = np.random.default_rng(seed)
    b = len(lens)
    max_pages = max(1, max(-(-n // page) for n in lens)) + 1
    need = [-(-n // page) for n in lens]
    n_pages = sum(need) + spare
    order = rng.permutation(n_pages)
    table = np.full((b, max_pages), -1, np.int32)
    at = 0
    for r, n in enumerate(need):
        table[r, :n] = order[at:at + n]
        at += n
    shape = (n_pages, kv, page, hd)
    codes = [rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2)]
    scale = [(np.exp(rng.standard_normal(shape[:2])) * s).astype(np.float32) for s in (0.01, 0.02)]
    for s in scale:
        s[order[at:]] = np.nan  # pages that nobody holds
    q_start = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    q = rng.standard_normal((int(q_start[-1]), kv * grp, hd)).astype(np.float32)
    if outlier and q.size:
        q[..., 0] *= 8
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    q = torch.from_numpy(q).to(t)
    return {"dtype": dtype, "q": q, "codes": codes, "scale": scale, "table": table, "lens": list(lens),
            "q_start": q_start, "n_new": max(list(new) + [1]), "hd": hd}


def run(torch, c, window=0, scale=None, max_new=None, max_len=None, place=None, stream=None, calls=1):
    dev = [torch.from_numpy(x).cuda() for x in c["codes"] + c["scale"]]
    ints = lambda z: torch.tensor(np.asarray(z, np.int32)).cuda()  # noqa: E731
    q = c["q"].cuda()
    out = torch.full_like(q, float("nan"))
    if place:
        q, out = place(q), place(out)
    scale = c["hd"] ** -0.5 if scale is None else scale
    a = jk.attn_q8_args(q, out, ints(c["q_start"]), ints(c["lens"]), ints(c["table"]),
                        c["n_new"] if max_new is None else max_new,
                        max(c["lens"]) if max_len is None else max_len, scale, window)
    cache = jk.kv_q8(*dev)
    n = jk.attn_q8_workspace_bytes(cache, a)
    ws = torch.full((max(16, n),), 0xFF, dtype=torch.uint8, device="cuda")  # (any content: NaN)
    torch.cuda.synchronize()
    for _ in range(calls):
        jk.dev_attn_q8(cache, a, ws, stream=stream)
    torch.cuda.synchronize()
    return out.float().cpu().numpy().astype(np.float64)


def check(torch, c, window=0, scale=None, **kw):
    got = run(torch, c, window, scale, **kw)
    want, bound = R.attention(c["q"].float().numpy(), *c["codes"], *c["scale"], c["q_start"], c["lens"], c["table"],
                              c["hd"] ** -0.5 if scale is None else scale, window, UNIT[c["dtype"]])
    far = np.abs(got - want)
    if c["dtype"] == "f16":  # a result past f16's largest value (65504; from 65520 on it rounds up) is infinite
        far[(np.abs(want) + bound >= 65520) & np.isinf(got) & (np.sign(got) == np.sign(want))] = 0
    assert np.all(far <= bound + 1e-30), (float(np.nanmax(far / (bound + 1e-30))), bool(np.isnan(got).any()))
    return got


DTYPES = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [16, 64, 80, 128, 144, 256])
def test_single_tokens(gpu, dtype, hd):
    """Decode steps: contexts of one token up to several pages, ends inside a tile, several group sizes."""
    for i, (kv, grp, page) in enumerate([(1, 1, 16), (2, 3, 64), (1, 8, 32), (1, 17, 16)]):
        lens = [1, 2, 15, 16, 17, 33, 130, 300]
        check(gpu, case(gpu, dtype, lens, [1] * len(lens), page, kv, grp, hd, seed=hd + i))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_ragged_prompts(gpu, dtype, page):
    """Chunks of prompts beside single tokens and requests that wait, of odd sizes."""
    lens, new = [5, 200, 40, 90, 1, 0, 77], [5, 37, 1, 0, 1, 0, 70]
    check(gpu, case(gpu, dtype, lens, new, page, 2, 4, 64, seed=page))
    check(gpu, case(gpu, dtype, lens, new, page, 1, 5, 96, seed=page + 1))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 7, 16, 33, 100])
def test_window(gpu, dtype, window):
    check(gpu, case(gpu, dtype, [3, 150, 90, 260], [1, 20, 1, 130], 32, 2, 2, 64, seed=window), window=window)


@pytest.mark.parametrize("dtype", DTYPES)
def test_long_context_split_over_workgroups(gpu, dtype):
    """One request over many workgroups: whole ones, a short last one, short requests beside it."""
    check(gpu, case(gpu, dtype, [3000], [1], 64, 1, 4, 128, seed=1))
    check(gpu, case(gpu, dtype, [2561, 1, 700], [1, 1, 2], 16, 2, 2, 64, seed=2))
    check(gpu, case(gpu, dtype, [1500], [3], 32, 1, 8, 80, seed=3), window=900)
    check(gpu, case(gpu, dtype, [1800], [60], 32, 1, 2, 128, seed=4))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_split_rows_among_many_requests(gpu, dtype, hd):
    """Long requests beside many short ones, some without new tokens: the joining finds each token's request."""
    lens = [1 + i % 30 for i in range(100)] + [2700, 5, 2100]
    new = [i % 3 // 2 for i in range(100)] + [2, 0, 1]
    check(gpu, case(gpu, dtype, lens, new, 64, 1, 4, hd, seed=6))
    check(gpu, case(gpu, dtype, lens[66:], new[66:], 16, 1, 20, hd, seed=7))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64), (256, 32)])
def test_long_prompts_split_over_workgroups(gpu, dtype, hd, page):
    """Chunks of prompts whose keys several workgroups share, beside a single token and a request of a few."""
    check(gpu, case(gpu, dtype, [1500, 1100, 70], [263, 1, 9], page, 1, 8, hd, seed=3))
    check(gpu, case(gpu, dtype, [2111], [257], page, 1, 8, hd, seed=4))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64), (96, 32)])
def test_many_prompts(gpu, dtype, hd, page):
    """So many columns that a workgroup takes the most of them, requests that end inside its tiles, and short ones."""
    kv, grp = (4, 32) if dtype == "f32" else (8, 16)
    lens = [65 + 9 * i for i in range(16)]
    new = [65, 65, 1, 33] * 4
    check(gpu, case(gpu, dtype, lens, new, page, kv, grp, hd, seed=5))


@pytest.mark.parametrize("dtype", DTYPES)
def test_bounds_that_are_off_do_not_change_results(gpu, dtype):
    """max_len is a matter of speed: too small and too large a one give the same within rounding."""
    c = case(gpu, dtype, [900, 20], [1, 1], 32, 1, 4, 64, seed=5)
    for n in (1, 64, 900, 100000):
        check(gpu, c, max_len=n)
    c = case(gpu, dtype, [300, 20], [40, 3], 32, 1, 4, 64, seed=6)
    check(gpu, c, max_new=300)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_see_nothing_and_pages_that_are_missing(gpu, dtype):
    """Lengths shorter than the step (its first queries stand before the cache), and table entries that are no pages:
    their tokens are as if not there, and rows left with nothing are 0."""
    c = case(gpu, dtype, [4, 0, 50], [7, 3, 2], 16, 1, 2, 64, seed=7)
    got = check(gpu, c)
    assert not got[:3].any() and not got[7:10].any()
    c = case(gpu, dtype, [60, 16], [2, 1], 16, 2, 2, 64, seed=8)
    c["table"][0, 1], c["table"][0, 3], c["table"][1, 0] = -1, 10 ** 6, -5
    got = check(gpu, c)
    assert not got[2].any()


def test_more_new_tokens_than_said(gpu):
    """Queries past max_new are left or computed, never wrong; the others are as ever."""
    torch = gpu
    c = case(torch, "f32", [100], [40], 16, 1, 2, 64, seed=9)
    whole, part = run(torch, c), run(torch, c, max_new=9)
    assert np.array_equal(whole[:9], part[:9]) or np.allclose(whole[:9], part[:9], atol=1e-5)
    rest = part[9:]
    assert np.all(np.isnan(rest) | (np.abs(rest - whole[9:]) < 1e-5))


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides_and_alignment(gpu, dtype):
    torch = gpu
    c = case(torch, dtype, [40, 200], [1, 33], 16, 2, 3, 80, seed=10)
    n, heads, hd = c["q"].shape
    base = check(torch, c)
    for wide, head, at in ((heads * hd * 2, hd, 0), (heads * hd + 5, hd, 1), (hd, n * hd, 0), (heads * (hd + 1), hd + 1, 3)):
        def place(x):
            buf = torch.full((n * heads * (hd + 1) * 3 + 16,), 3.0, dtype=x.dtype, device="cuda")
            y = torch.as_strided(buf, (n, heads, hd), (wide, head, 1), at)
            y.copy_(x)
            return y
        assert np.array_equal(check(torch, c, place=place), base)


@pytest.mark.parametrize("dtype", DTYPES)
def test_extreme_values(gpu, dtype):
    """One key that takes all the weight, scores that are all equal, scales far apart, zero queries and pages of zeros."""
    torch = gpu
    c = case(torch, dtype, [100, 70], [1, 40], 16, 1, 2, 64, seed=11)
    check(torch, c, scale=20.0)
    check(torch, c, scale=0.0)
    check(torch, c, scale=-1.0)
    c["q"][0] = 0
    c["scale"][1][c["table"][0, 2]] = 0
    c["scale"][0][c["table"][1, 0]] = 0
    check(torch, c)
    c["scale"][1][c["table"][0, 1]] *= 1e6
    c["scale"][1][c["table"][1, 3]] *= 1e-6
    check(torch, c)
    c["scale"][0][c["table"][0, 0]] *= 1e-3
    check(torch, c)


def test_queries_of_any_size(gpu):
    """Rows of very large and very small f32 queries keep their precision (each row is brought to f16's range)."""
    torch = gpu
    c = case(torch, "f32", [90, 70], [1, 20], 16, 1, 2, 64, seed=12)
    for f in (1e-37, 1e-30, 1e-10, 1e10, 1e30):
        d = dict(c, q=c["q"] * f)
        check(torch, d, scale=64 ** -0.5 / f)


def test_a_query_that_is_not_a_number_keeps_to_its_row(gpu):
    torch = gpu
    c = case(torch, "f32", [90, 1500], [5, 1], 16, 1, 2, 64, seed=13)
    want = run(torch, c)
    c["q"][2, 1, 7] = float("nan")
    c["q"][5, 0, 0] = float("nan")
    got = run(torch, c)
    bad = np.zeros(got.shape[:2], bool)
    bad[2, 1] = bad[5, 0] = True
    assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], want[~bad])


def test_on_another_stream_and_in_a_graph(gpu):
    torch = gpu
    c = case(torch, "bf16", [1300, 40, 7], [1, 1, 1], 64, 2, 4, 128, seed=14)
    want = run(torch, c)
    s = torch.cuda.Stream()
    assert np.array_equal(run(torch, c, stream=s.cuda_stream, calls=3), want)
    dev = [torch.from_numpy(x).cuda() for x in c["codes"] + c["scale"]]
    ints = lambda z: torch.tensor(np.asarray(z, np.int32)).cuda()  # noqa: E731
    q, out = c["q"].cuda(), torch.zeros_like(c["q"].cuda())
    a = jk.attn_q8_args(q, out, ints(c["q_start"]), ints(c["lens"]), ints(c["table"]), 1, 1300, 128 ** -0.5)
    cache = jk.kv_q8(*dev)
    ws = torch.empty(max(16, jk.attn_q8_workspace_bytes(cache, a)), dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        jk.dev_attn_q8(cache, a, ws, stream=s.cuda_stream)
    for i in range(5):
        out.fill_(float(i))
        ws.fill_(i)
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.float().cpu().numpy().astype(np.float64), want)
        q2 = torch.randn(64, 64, device="cuda") @ torch.randn(64, 64, device="cuda")
        assert bool(torch.isfinite(q2).all())


def test_the_same_bits_every_time(gpu):
    torch = gpu
    c = case(torch, "f32", [3000, 500], [1, 2], 64, 2, 4, 64, seed=15)
    want = run(torch, c)
    for _ in range(3):
        assert np.array_equal(run(torch, c), want)
