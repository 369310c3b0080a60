"""Whose a page is, on the GPU: steps that are dropped, releases and reorderings in random order against a plain implementation.

Tables, owners, lengths, the stack and what every row then reads are compared exactly after every call.
"""
import numpy as np
import pytest

import jk
import paged_owners as O

pytestmark = pytest.mark.gpu


class Dev:
    """The device's side of a batch, with a cache whose codes say which token a place holds."""

    def __init__(self, torch, b, max_pages, n_pages, page, cap):
        ints = lambda *n: torch.full(n, -7, dtype=torch.int32, device="cuda")  # noqa: E731
        self.torch, self.page = torch, page
        self.lens, self.table, self.owned = ints(b), ints(b, max_pages), ints(b, max_pages)
        self.free, self.n_free, self.status = ints(n_pages), ints(1), ints(1)
        self.apart = ints(b), ints(1)
        self.q_start, self.out = ints(b + 1), [ints(cap) for _ in range(3)]
        self.p = jk.paged(self.lens, self.table, self.owned, self.free, self.n_free, page)
        self.step = jk.paged_step(self.q_start, *self.out, self.status)
        self.codes = [torch.zeros((n_pages, 1, page, 16), dtype=torch.int8, device="cuda") for _ in range(2)]
        self.scales = [torch.ones((n_pages, 1), device="cuda") for _ in range(2)]
        self.cache = jk.kv_q8(*self.codes, *self.scales)
        jk.dev_paged_reset(self.p)

    def dev(self, x):
        return self.torch.tensor(np.asarray(x, np.int32)).cuda()

    def extend(self, n_new, drop=False):
        jk.dev_paged_extend(self.p, self.dev(n_new), self.step, *(self.apart if drop else ()))
        n = int(self.q_start[-1])
        return (int(self.status),) + tuple(x.tolist()[:n] for x in self.out)

    def write(self, slots, first):
        """Token first + i into slots[i], in keys and values."""
        if not slots:
            return
        t = np.arange(first, first + len(slots))
        code = np.stack([t % 127, t // 127 % 127, t // 16129 % 127], 1).astype(np.int8)
        s = self.torch.tensor(np.asarray(slots), device="cuda")
        for x, flip in zip(self.codes, (1, -1)):
            x.view(-1, 16)[s, :3] = self.torch.from_numpy(code * flip).cuda().to(self.torch.int8)

    def reorder(self, parent, width):
        q = self.dev(parent)
        jk.dev_paged_reorder(self.p, q, width, self.status)
        jk.dev_kv_reorder_q8(self.cache, self.p, q, width, self.status)
        return int(self.status)

    def same(self, ref, held):
        assert self.lens.tolist() == ref.lens
        assert np.array_equal(self.table.cpu().numpy()[:, :], ref.table)
        assert np.array_equal(self.owned.cpu().numpy(), ref.owned)
        assert int(self.n_free) == ref.height and self.free.tolist()[:ref.height] == [int(x) for x in ref.free]
        for x, flip in zip(self.codes, (1, -1)):
            c = x.cpu().numpy().reshape(-1, self.page, 16)[..., :3].astype(np.int64) * flip
            c = c[..., 0] + 127 * c[..., 1] + 16129 * c[..., 2]
            for r, tokens in enumerate(held.rows):
                t = np.arange(len(tokens))
                assert np.array_equal(c[ref.table[r, t // self.page], t % self.page], tokens), f"row {r}"


def both(d, p, h, width, calls, check=True):
    """Carries out the calls on both sides; the kernels' outputs are the plain implementation's."""
    for what, x in calls:
        if what == "release":
            jk.dev_paged_release(d.p, d.dev(x))
            p.release(x)
            h.release(x)
        elif what == "reorder":
            st, moves = p.reorder(x, width)
            assert d.reorder(x, width) == st
            if st == 0:
                h.reorder(x, width, moves)
        else:
            want = p.extend(x, drop=what == "draft")
            assert d.extend(x, drop=what == "draft") == want
            if what == "draft":  # (a dropped step's tokens are written before it is dropped)
                if want[0] == 0:
                    assert d.apart[0].tolist() == [a + n for a, n in zip(p.lens, x)]
            d.write(want[1], h.next)
            h.write(want[1], want[3], keep=what == "extend")
        d.same(p, h)
        if check:
            O.check(p, h, width)


@pytest.mark.parametrize("unequal,drafts", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("groups,width,max_pages,n_steps", [(1, 1, 8, 30), (1, 4, 8, 40), (3, 8, 12, 30), (2, 13, 8, 20),
                                                            (90, 4, 12, 8), (1, 32, 1030, 8)])
def test_random_sequences(gpu, groups, width, max_pages, n_steps, unequal, drafts):
    for seed in range(2):
        rng = np.random.default_rng(seed)
        b, n_pages = groups * width, groups * width * min(max_pages, 7)
        d = Dev(gpu, b, max_pages, n_pages, 16, b * 70)
        p, h = O.Owners(b, max_pages, n_pages, 16), O.Held(b, n_pages, 16)
        both(d, p, h, width, O.steps(rng, groups, width, 16, max_pages, n_steps, unequal, drafts), check=b <= 32)


@pytest.mark.parametrize("drafts", [False, True])
@pytest.mark.parametrize("groups,width", [(300, 4), (206, 5), (75, 16)])
def test_batches_of_several_passes(gpu, groups, width, drafts):
    """More requests than the planning workgroup takes at once."""
    rng = np.random.default_rng(3)
    b, n_pages = groups * width, groups * width * 5
    d = Dev(gpu, b, 9, n_pages, 16, b * 40)
    p, h = O.Owners(b, 9, n_pages, 16), O.Held(b, n_pages, 16)
    both(d, p, h, width, O.steps(rng, groups, width, 16, 9, 4, True, drafts), check=False)


def test_dropped_step_then_release(gpu):
    """The pages of a dropped step are free again, whoever gets them next: no page has two owners or is free twice."""
    d, p, h = Dev(gpu, 3, 8, 12, 16, 64), O.Owners(3, 8, 12, 16), O.Held(3, 12, 16)
    both(d, p, h, 1, [("extend", [16, 16, 0]), ("draft", [5, 0, 0]), ("extend", [0, 1, 0]), ("release", [1, 0, 0]),
                      ("extend", [0, 0, 40]), ("release", [0, 1, 1])])
    assert sorted(d.free.tolist()) == list(range(12)) and int(d.n_free) == 12


def test_dropped_step_then_release_of_one_table(gpu):
    """The same where table and owned are one array."""
    torch = gpu
    d = Dev(torch, 2, 4, 6, 16, 64)
    d.p = jk.paged(d.lens, d.table, d.table, d.free, d.n_free, 16)
    jk.dev_paged_reset(d.p)
    d.extend([16, 16])
    d.extend([20, 0], drop=True)
    d.extend([0, 1])
    assert int(d.n_free) == 3
    jk.dev_paged_release(d.p, d.dev([1, 0]))
    assert int(d.n_free) == 4
    in_use = set(d.table[1, :2].tolist())
    assert len(in_use) == 2 and sorted(d.free.tolist()[:4] + list(in_use)) == list(range(6))


def test_dropped_step_then_reordering(gpu):
    """A page that a dropped step left in a row's place is not the row's to fill: another request may have it."""
    d, p, h = Dev(gpu, 4, 4, 16, 16, 64), O.Owners(4, 4, 16, 16), O.Held(4, 16, 16)
    both(d, p, h, 2, [("extend", [16, 0, 20, 0]), ("reorder", [0, 0, 0, 0]), ("draft", [4, 4, 0, 0]),
                      ("extend", [0, 0, 16, 16]), ("draft", [0, 30, 0, 0]), ("extend", [3, 0, 0, 0]), ("reorder", [0, 0, 1, 0]),
                      ("release", [1, 1, 0, 0]), ("extend", [0, 0, 5, 5]), ("release", [0, 0, 1, 1])])
    assert int(d.n_free) == 16


@pytest.mark.parametrize("lens,parents", [([17, 15], [1, 0]), ([16, 15], [1, 0]), ([33, 20, 20], [1, 0, 2])])
@pytest.mark.parametrize("max_pages", [4, 1100])
def test_rows_that_would_go_back_to_fewer_full_pages(gpu, lens, parents, max_pages):
    """A full page can be shared, so its owner must not fill it again: a status, and nothing changes."""
    torch = gpu
    w = len(lens)
    d, p, h = Dev(torch, w, max_pages, 16, 16, 80), O.Owners(w, max_pages, 16, 16), O.Held(w, 16, 16)
    both(d, p, h, w, [("extend", lens), ("reorder", parents)])
    assert p.reorder(parents, w)[0] == jk.PAGED_SHORTER
    lo, to = torch.empty_like(d.lens), torch.empty_like(d.table)
    jk.dev_paged_reorder(d.p, d.dev(parents), w, d.status, lo, to)
    assert int(d.status) == jk.PAGED_SHORTER and torch.equal(lo, d.lens) and torch.equal(to, d.table)
    both(d, p, h, w, [("extend", [1] * w)])


@pytest.mark.parametrize("cap", [64, 9000])
def test_pages_that_a_row_went_back_from(gpu, cap):
    """To the first token of the page it was filling: the page stays the row's and is begun again, without another."""
    d, p, h = Dev(gpu, 2, 4, 8, 16, cap), O.Owners(2, 4, 8, 16), O.Held(2, 8, 16)
    both(d, p, h, 2, [("extend", [20, 16]), ("reorder", [1, 0]), ("draft", [3, 0]), ("extend", [2, 0]), ("extend", [16, 9]),
                      ("draft", [9, 9]), ("reorder", [0, 1]), ("release", [1, 1])])
    assert int(d.n_free) == 8


def test_lengths_out_of_range(gpu):
    """A row's own length is checked before its places are looked at, also where its parent's is in range."""
    torch = gpu
    for bad in (-1, 4 * 16 + 1, 2 ** 31 - 1):
        d, p, h = Dev(torch, 2, 4, 8, 16, 64), O.Owners(2, 4, 8, 16), O.Held(2, 8, 16)
        both(d, p, h, 2, [("extend", [20, 0])])
        d.lens[1] = bad
        assert d.reorder([0, 0], 2) == jk.PAGED_BAD_LENGTH
        assert d.lens.tolist() == [20, bad] and int(d.n_free) == 6
