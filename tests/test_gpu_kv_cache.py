"""The 8-bit attention cache on the GPU: storing, reading back and moving pages.

Codes and scales follow an f32 recipe of single roundings (a division by 127, one reciprocal, a product and a rounding to the
nearest integer), so they are compared exactly with the same recipe in numpy.
"""
import numpy as np
import pytest

import jk
import paged_ref as R

pytestmark = pytest.mark.gpu


def values(rng, shape, dtype):
    x = rng.standard_normal(shape).astype(np.float32) * np.exp(rng.standard_normal(shape[0]))[:, None, None]
    if dtype == "f16":
        return x.astype(np.float16).astype(np.float32)
    if dtype == "bf16":
        b = x.astype(np.float32).view(np.uint32)
        return ((b + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return x.astype(np.float32)


class Cache:
    def __init__(self, torch, n_pages, kv, page, hd, seed=0):
        rng = np.random.default_rng(seed)
        self.torch = torch
        shape = (n_pages, kv, page, hd)
        self.host = [rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2)]
        self.scale = [np.exp(rng.standard_normal(shape[:2]) * 2).astype(np.float32) for _ in range(2)]
        self.dev = [torch.from_numpy(x.copy()).cuda() for x in self.host + self.scale]
        self.c = jk.kv_q8(*self.dev)

    def append(self, k, v, slots, dtype, stream=None, place=None):
        torch = self.torch
        t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
        dk, dv = (torch.from_numpy(x).cuda().to(t) for x in (k, v))
        if place:
            dk, dv = place(dk), place(dv)
        jk.dev_kv_append_q8(self.c, dk, dv, torch.tensor(slots, dtype=torch.int32).cuda(), stream=stream)
        for i, x in enumerate((k, v)):
            R.append(self.host[i], self.scale[i], x, slots)

    def same(self):
        got = [x.cpu().numpy() for x in self.dev]
        for i in range(2):
            assert np.array_equal(got[2 + i], self.scale[i], equal_nan=True)
            assert np.array_equal(got[i], self.host[i])


def slots_of(page, runs):
    """Slots of runs (page id, first row, tokens)."""
    return [p * page + row + i for p, row, n in runs for i in range(n)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("page,kv,hd", [(16, 1, 16), (16, 3, 80), (64, 2, 128), (128, 1, 96), (256, 1, 256)])
def test_append(gpu, dtype, page, kv, hd):
    """Whole pages, begun ones that go on, single tokens at every kind of row, and skipped slots."""
    rng = np.random.default_rng(page + hd)
    c = Cache(gpu, 9, kv, page, hd)
    half = page // 2
    runs = [(3, 0, page), (5, 0, half), (0, 0, 1), (7, page - 1, 1), (2, 3, 5)]
    slots = slots_of(page, runs)
    c.append(values(rng, (len(slots), kv, hd), dtype), values(rng, (len(slots), kv, hd), dtype), slots, dtype)
    c.same()
    slots = slots_of(page, [(5, half, half)]) + [-1, 9 * page, -5] + slots_of(page, [(0, 1, 1), (2, 8, 1)]) + [-1]
    for _ in range(3):  # (the same rows again, with other values: scales only grow)
        c.append(values(rng, (len(slots), kv, hd), dtype), values(rng, (len(slots), kv, hd), dtype), slots, dtype)
        c.same()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_append_of_many_tokens(gpu, dtype):
    """More tokens than a step of single-token workgroups takes: whole pages a workgroup, runs across its bounds."""
    rng = np.random.default_rng(5)
    page, kv, hd = 32, 2, 64
    c = Cache(gpu, 60, kv, page, hd)
    order = rng.permutation(60)
    runs = [(int(p), 0, page) for p in order[:30]] + [(int(order[30]), 5, 27), (int(order[31]), 0, 13)]
    runs += [(int(p), 7, 3) for p in order[32:50]]
    slots = slots_of(page, runs) + [-1] * 40
    assert len(slots) > 1024
    c.append(values(rng, (len(slots), kv, hd), dtype), values(rng, (len(slots), kv, hd), dtype), slots, dtype)
    c.same()


def test_append_token_by_token_stays_close(gpu):
    """A page filled by single tokens: every value within half a step of its own scale plus half a step of
    each rescaling since (each rescaled code is rounded once, with the new, larger scale)."""
    rng = np.random.default_rng(9)
    page, hd = 64, 64
    c = Cache(gpu, 2, 1, page, hd)
    x = values(rng, (page, 1, hd), "f32")
    x *= np.linspace(0.2, 4, page)[:, None, None].astype(np.float32)
    allowed, d, n = np.zeros(page), 0.0, 0
    for t in range(page):
        c.append(x[t:t + 1], x[t:t + 1], [page + t], "f32")
        new = float(c.scale[0][1, 0])
        if new > d:
            allowed[:t] += new / 2
            n += 1
        d = new
        allowed[t] = new / 2
    c.same()
    assert 4 < n < page
    got = c.dev[0].cpu().numpy()[1, 0].astype(np.float64) * d
    assert np.all(np.abs(got - x[:, 0]) <= (allowed * (1 + 1e-5))[:, None])


def test_values_that_are_not_finite_or_tiny(gpu):
    c = Cache(gpu, 4, 1, 16, 16)
    x = np.ones((4, 1, 16), np.float32)
    x[0, 0, :4] = [np.nan, np.inf, -np.inf, -3]
    x[1] = np.nan
    x[2] = 2.0 ** -120
    x[3] = 2.0 ** -118
    c.append(x, -x, [0, 16, 32, 48], "f32")
    c.same()
    k = c.dev[0].cpu().numpy()
    assert k[0, 0, 0, :5].tolist() == [0, 0, 0, -127, 42]
    assert not k[1, 0, 0].any() and not k[2, 0, 0].any() and (k[3, 0, 0] == 127).all()
    assert c.dev[2].cpu().numpy()[:, 0].tolist()[1:3] == [0, 0]
    # a page of zeros goes on with other values, and one whose stored scale is not a number
    c.dev[2][2, 0] = c.scale[0][2, 0] = np.nan
    y = np.full((2, 1, 16), 5, np.float32)
    c.append(y, y, [17, 33], "f32")
    c.same()
    assert not c.dev[0][1:3, 0, 0].any()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_append_strided_and_unaligned(gpu, dtype):
    """Keys and values inside wider rows, and one element past a 16-byte boundary."""
    torch = gpu
    rng = np.random.default_rng(11)
    page, kv, hd, n = 16, 2, 48, 21
    slots = slots_of(page, [(1, 0, 16), (2, 0, 5)])
    for wide, at in ((3 * kv * hd, 0), (3 * kv * hd + 3, 1)):
        def place(x):
            buf = torch.zeros(n * wide + 8, dtype=x.dtype, device="cuda")
            y = torch.as_strided(buf, (n, kv, hd), (wide, hd, 1), at)
            y.copy_(x)
            return y
        c = Cache(torch, 4, kv, page, hd, seed=at)
        c.append(values(rng, (n, kv, hd), dtype), values(rng, (n, kv, hd), dtype), slots, dtype, place=place)
        c.same()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_read(gpu, dtype):
    torch = gpu
    t = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    c = Cache(torch, 5, 3, 32, 80)
    slots = [7, 0, 5 * 32 - 1, -1, 5 * 32, 64, 64, 2 ** 31 - 1]
    k = torch.full((len(slots), 3, 80), 9.0, dtype=t, device="cuda")
    v = torch.full_like(k, 9.0)
    s = torch.tensor(slots, dtype=torch.int32).cuda()
    jk.dev_kv_read_q8(c.c, s, k, v)
    for i, out in enumerate((k, v)):
        want = np.zeros((len(slots), 3, 80), np.float32)
        for j, x in enumerate(slots):
            if 0 <= x < 160:
                want[j] = c.host[i][x // 32, :, x % 32].astype(np.float32) * c.scale[i][x // 32][:, None]
        assert torch.equal(out.cpu(), torch.from_numpy(want).to(t))
    one = torch.full_like(k, 9.0)
    jk.dev_kv_read_q8(c.c, s, None, one)
    assert torch.equal(one, v)
    # an output one element past a 16-byte boundary
    buf = torch.zeros(len(slots) * 240 + 1, dtype=t, device="cuda")
    jk.dev_kv_read_q8(c.c, s, buf[1:], None)
    assert torch.equal(buf[1:].view_as(k), k)


def test_places_past_32_bits(gpu):
    """Codes past 4 GiB of a cache, appended, read back and attended to."""
    torch = gpu
    page, kv, hd = 256, 4, 256
    n_pages = (1 << 32) // (page * kv * hd) + 40
    k = torch.empty((n_pages, kv, page, hd), dtype=torch.int8, device="cuda")
    v = torch.empty_like(k)
    scales = [torch.ones((n_pages, kv), device="cuda") for _ in range(2)]
    c = jk.kv_q8(k, v, *scales)
    rng = np.random.default_rng(3)
    x = [torch.from_numpy(values(rng, (300, kv, hd), "f32")).cuda() for _ in range(2)]
    pages = [n_pages - 1, n_pages - 3]
    slots = torch.tensor(slots_of(page, [(pages[0], 0, 256), (pages[1], 0, 44)]), dtype=torch.int32).cuda()
    jk.dev_kv_append_q8(c, x[0], x[1], slots)
    out = [torch.empty((300, kv, hd), device="cuda") for _ in range(2)]
    jk.dev_kv_read_q8(c, slots, *out)
    small = Cache(torch, 2, kv, page, hd)
    small.append(x[0].cpu().numpy(), x[1].cpu().numpy(), list(range(300)), "f32")
    want = [torch.empty_like(out[0]) for _ in range(2)]
    jk.dev_kv_read_q8(small.c, torch.arange(300, dtype=torch.int32).cuda(), *want)
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
    q = torch.randn((1, 8, hd), device="cuda")
    y = [torch.empty_like(q) for _ in range(2)]
    for cache, table, o in ((c, pages, y[0]), (small.c, [0, 1], y[1])):
        ints = lambda z: torch.tensor(z, dtype=torch.int32).cuda()  # noqa: E731
        a = jk.attn_q8_args(q, o, ints([0, 1]), ints([300]), ints([table]), 1, 300, hd ** -0.5)
        ws = torch.empty(max(16, jk.attn_q8_workspace_bytes(cache, a)), dtype=torch.uint8, device="cuda")
        jk.dev_attn_q8(cache, a, ws)
    assert torch.equal(*y)


@pytest.mark.parametrize("width,hd", [(2, 64), (8, 128), (13, 16), (32, 48)])
def test_reorder_moves_the_open_pages(gpu, width, hd):
    torch = gpu
    page, kv, groups = 32, 2, 3
    rng = np.random.default_rng(width)
    b, n_pages = width * groups, width * groups * 4
    c = Cache(torch, n_pages, kv, page, hd)
    ref = R.Pages(b, 4, n_pages, page)
    n = rng.integers(page, 2 * page, b)
    ref.extend(list(n), int(n.sum()))
    ints = lambda z: torch.tensor(np.asarray(z, np.int32)).cuda()  # noqa: E731
    free = np.full(n_pages, -1)
    free[:len(ref.free)] = ref.free
    lens, table, owned, stack, height = ints(ref.lens), ints(ref.table), ints(ref.owned), ints(free), ints([len(ref.free)])
    p = jk.paged(lens, table, owned, stack, height, page)
    status = ints([-7])
    for i in range(3):
        parent = rng.integers(0, width, b)
        jk.dev_paged_reorder(p, ints(parent), width, status)
        jk.dev_kv_reorder_q8(c.c, p, ints(parent), width, status)
        st, moves = ref.reorder(list(parent), width)
        assert st == int(status) == 0
        old = [x.copy() for x in c.host + c.scale]
        for src, dst, rows in moves:
            for k in range(2):
                c.host[k][dst, :, :rows] = old[k][src, :, :rows]
                c.scale[k][dst] = old[2 + k][src]
        # (16-byte pieces: only whole rows move)
        c.same()
    # where the tables' reordering was refused nothing moves
    status.fill_(jk.PAGED_NO_PAGES)
    jk.dev_kv_reorder_q8(c.c, p, ints(np.roll(np.arange(b) % width, 1)), width, status)
    c.same()
