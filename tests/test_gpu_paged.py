"""Pages of a batch's attention cache on the GPU: plans, releases and reorderings against a plain implementation.

All outputs are integers and compared exactly.
"""
import numpy as np
import pytest

import jk
import paged_ref as R

pytestmark = pytest.mark.gpu


class Dev:
    """The device arrays of a batch and of a step."""

    def __init__(self, torch, b, max_pages, n_pages, page, cap, apart=True):
        ints = lambda *n: torch.full(n, -7, dtype=torch.int32, device="cuda")  # noqa: E731
        self.torch = torch
        self.lens, self.table, self.free, self.n_free = ints(b), ints(b, max_pages), ints(n_pages), ints(1)
        self.owned = ints(b, max_pages) if apart else self.table
        self.p = jk.paged(self.lens, self.table, self.owned, self.free, self.n_free, page)
        self.step_of(cap, b)
        jk.dev_paged_reset(self.p)

    def step_of(self, cap, b):
        ints = lambda n: self.torch.full((n,), -7, dtype=self.torch.int32, device="cuda")  # noqa: E731
        self.out = [ints(b + 1), ints(cap), ints(cap), ints(cap), ints(1)]
        self.step = jk.paged_step(*self.out)

    def dev(self, x):
        return self.torch.tensor(np.asarray(x, np.int32)).cuda()

    def same(self, ref):
        assert self.lens.tolist() == ref.lens
        assert np.array_equal(self.table.cpu().numpy(), ref.table)
        if self.owned is not self.table:
            assert np.array_equal(self.owned.cpu().numpy(), ref.owned)
        n = int(self.n_free)
        assert n == len(ref.free) and self.free.tolist()[:n] == ref.free

    def extend(self, ref, n_new, **kw):
        cap = self.step.max_tokens
        jk.dev_paged_extend(self.p, self.dev(n_new), self.step, **kw)
        want = ref.extend(list(n_new), cap)
        got = [x.tolist() for x in self.out]
        assert got[4] == [want[0]]
        assert got[0] == want[1] and got[1] == want[2] and got[2] == want[3] and got[3] == want[4]
        return want[0]


@pytest.mark.parametrize("b,page,cap", [(1, 16, 1), (3, 16, 70), (64, 64, 2048), (5, 256, 3000), (1024, 32, 2500),
                                        (1025, 16, 2048), (2500, 16, 6001), (7, 64, 8193), (2500, 16, 9000)])
def test_extend_and_release(gpu, b, page, cap):
    rng = np.random.default_rng(b + page)
    max_pages = 12
    d, ref = Dev(gpu, b, max_pages, max(24, 4 * b), page, cap, apart=b % 2 == 0), None
    ref = R.Pages(b, max_pages, max(24, 4 * b), page)
    for i in range(6):
        n = rng.integers(0, 3, b)
        n[rng.integers(0, b)] += rng.integers(0, 3 * page)
        n = np.minimum(n, 12 * page - np.array(ref.lens))
        over = np.cumsum(n) > cap
        n[over] = 0
        d.extend(ref, n)
        d.same(ref)
        ended = rng.integers(0, 4, b) == 0
        jk.dev_paged_release(d.p, d.dev(ended))
        ref.release(ended)
        d.same(ref)


def test_extend_of_nothing_and_of_whole_pages(gpu):
    d, ref = Dev(gpu, 4, 8, 40, 16, 64), R.Pages(4, 8, 40, 16)
    for n in ([0, 0, 0, 0], [16, 0, 16, 1], [16, 16, 0, 15], [0, 0, 0, 0], [1, 0, 1, 0]):
        assert d.extend(ref, n) == 0
        d.same(ref)


def test_extend_out_of_place_leaves_the_old_state(gpu):
    """A tentative step: the old lengths and stack height stay, and going on from them gives the same pages again."""
    torch = gpu
    d, ref = Dev(torch, 3, 8, 20, 16, 40), R.Pages(3, 8, 20, 16)
    d.extend(ref, [5, 16, 9])
    lens, height = d.lens.clone(), d.n_free.clone()
    lo, fo = torch.empty_like(lens), torch.empty_like(height)
    jk.dev_paged_extend(d.p, d.dev([12, 1, 0]), d.step, lo, fo)
    assert torch.equal(d.lens, lens) and torch.equal(d.n_free, height)
    assert lo.tolist() == [17, 17, 9] and int(fo) == int(height) - 2
    first = [x.tolist() for x in d.out]
    assert d.extend(ref, [12, 1, 0]) == 0
    assert first == [x.tolist() for x in d.out]


@pytest.mark.parametrize("cap", [64, 5000, 8200])
def test_steps_that_do_not_fit_change_nothing(gpu, cap):
    d, ref = Dev(gpu, 3, 4, 5, 16, cap), R.Pages(3, 4, 5, 16)
    assert d.extend(ref, [20, 3, 0]) == 0
    for n, why in (([30, 14, 16], 1), ([45, 0, 0], 2), ([0, -1, 0], 3), ([2 ** 31 - 1, 2 ** 31 - 1, 0], 2)):
        assert d.extend(ref, n) == why
        d.same(ref)
    assert d.extend(ref, [28, 0, 0]) == 0
    d.lens[1] = 4 * 16 + 1  # a length that the table cannot hold
    ref.lens[1] = 4 * 16 + 1
    assert d.extend(ref, [0, 0, 1]) == 3


def test_step_of_more_tokens_than_asked_for(gpu):
    d, ref = Dev(gpu, 2, 8, 20, 16, 8), R.Pages(2, 8, 20, 16)
    assert d.extend(ref, [5, 4]) == 2
    assert d.extend(ref, [5, 3]) == 0
    d.same(ref)


def test_no_tokens_at_all(gpu):
    d, ref = Dev(gpu, 2, 8, 20, 16, 0), R.Pages(2, 8, 20, 16)
    assert d.extend(ref, [0, 0]) == 0
    d.same(ref)


@pytest.mark.parametrize("width,groups,page", [(1, 3, 16), (2, 5, 16), (4, 1, 32), (8, 3, 16), (9, 2, 16), (32, 2, 64),
                                               (5, 205, 16), (9, 120, 16)])
@pytest.mark.parametrize("in_place", [True, False])
def test_reorder(gpu, width, groups, page, in_place):
    """A prompt in the first row of each group, then steps of a token a row, each after a reordering."""
    torch = gpu
    b, max_pages = width * groups, 9
    rng = np.random.default_rng(width * 10 + groups)
    n_pages = b * max_pages
    d, ref = Dev(torch, b, max_pages, n_pages, page, b * 2 * page), R.Pages(b, max_pages, n_pages, page)
    n = np.zeros(b, np.int64)
    n[::width] = rng.integers(1, 2 * page, groups)
    assert d.extend(ref, n) == 0
    status = torch.full((1,), -7, dtype=torch.int32, device="cuda")
    for i in range(5):
        parent = np.zeros(b, np.int64) if i == 0 else rng.integers(0, width, b)
        if i == 2:
            parent[0] = width + 3  # out of range: goes on from itself
        if in_place:
            jk.dev_paged_reorder(d.p, d.dev(parent), width, status)
        else:
            lo, to = torch.empty_like(d.lens), torch.empty_like(d.table)
            jk.dev_paged_reorder(d.p, d.dev(parent), width, status, lo, to)
            d.lens.copy_(lo)
            d.table.copy_(to)
        st, _ = ref.reorder(list(parent), width)
        assert (int(status), st) == (0, 0)
        d.same(ref)
        assert d.extend(ref, [1 if i != 3 else page] * b) == 0
        d.same(ref)


def test_reorder_refusals_on_the_device(gpu):
    torch = gpu
    status = torch.full((1,), -7, dtype=torch.int32, device="cuda")
    d, ref = Dev(torch, 4, 4, 6, 16, 64), R.Pages(4, 4, 6, 16)
    d.extend(ref, [20, 20, 0, 0])  # 4 of 6 pages
    jk.dev_paged_reorder(d.p, d.dev([0, 0, 0, 1]), 4, status)
    assert int(status) == 0 and ref.reorder([0, 0, 0, 1], 4)[0] == 0
    d.same(ref)
    d, ref = Dev(torch, 4, 4, 5, 16, 64), R.Pages(4, 4, 5, 16)
    d.extend(ref, [20, 20, 0, 0])
    lo, to = torch.empty_like(d.lens), torch.empty_like(d.table)
    jk.dev_paged_reorder(d.p, d.dev([0, 0, 0, 1]), 4, status, lo, to)  # two pages needed, one free
    assert int(status) == jk.PAGED_NO_PAGES == ref.reorder([0, 0, 0, 1], 4)[0]
    d.same(ref)
    assert torch.equal(lo, d.lens) and torch.equal(to, d.table)
    d.owned[0, 1] = -1  # the open page of row 0 is no longer its own
    ref.owned[0, 1] = -1
    jk.dev_paged_reorder(d.p, d.dev([0, 1, 2, 3]), 4, status)
    assert int(status) == jk.PAGED_NOT_OWNED == ref.reorder([0, 1, 2, 3], 4)[0]
    d.same(ref)


def test_pages_out_of_range_give_no_slots(gpu):
    d, ref = Dev(gpu, 2, 4, 8, 16, 64), R.Pages(2, 4, 8, 16)
    d.extend(ref, [10, 10])
    d.table[0, 0] = 8  # not a page
    d.owned[0, 0] = 8
    jk.dev_paged_extend(d.p, d.dev([2, 2]), d.step)
    assert d.out[1].tolist()[:4] == [-1, -1] + [int(d.table[1, 0]) * 16 + 10, int(d.table[1, 0]) * 16 + 11]


def test_plan_in_a_graph(gpu):
    """A captured step replayed between eager ones."""
    torch = gpu
    d, ref = Dev(torch, 6, 16, 96, 16, 6), R.Pages(6, 16, 96, 16)
    d.extend(ref, [1] * 6)
    n = d.dev([1] * 6)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            jk.dev_paged_extend(d.p, n, d.step, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for i in range(20):
        g.replay()
        torch.cuda.synchronize()
        want = ref.extend([1] * 6, 6)
        assert [x.tolist() for x in d.out] == [want[1], want[2], want[3], want[4], [0]]
        d.same(ref)
        if i % 7 == 3:
            d.extend(ref, [1, 0, 1, 0, 1, 0])
