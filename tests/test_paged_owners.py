"""The plain implementation of the pages' ownership against a check that knows only what must hold (no GPU needed)."""
import numpy as np
import pytest

import paged_owners as O


def run(p, h, width, calls):
    """Carries out the calls on the plain implementation and on the contents; the statuses seen."""
    seen = []
    for what, x in calls:
        if what == "extend":
            st, slots, _, requests = p.extend(x)
            h.write(slots, requests)
        elif what == "draft":
            st, slots, _, requests = p.extend(x, drop=True)
            h.write(slots, requests, keep=False)
        elif what == "release":
            st = 0
            p.release(x)
            h.release(x)
        else:
            st, moves = p.reorder(x, width)
            if st == 0:
                h.reorder(x, width, moves)
        seen.append((what, st))
        O.check(p, h, width)
    return seen


@pytest.mark.parametrize("unequal", [False, True])
@pytest.mark.parametrize("groups,width", [(1, 1), (1, 2), (2, 3), (3, 4), (1, 8)])
def test_random_sequences(groups, width, unequal):
    went_back = 0
    for seed in range(12):
        rng = np.random.default_rng(seed)
        p = O.Owners(groups * width, 12, groups * width * 8, 4)
        seen = run(p, O.Held(groups * width, p.n_pages, 4), width, O.steps(rng, groups, width, 4, 12, 60, unequal))
        went_back += ("reorder", 5) in seen
        p.release([1] * (groups * width))
        assert sorted(p.free) == list(range(p.n_pages))
    assert unequal and width > 1 or not went_back


def test_dropped_step_then_release():
    """The pages of a dropped step are free again, whoever gets them next."""
    p, h = O.Owners(3, 8, 12, 16), O.Held(3, 12, 16)
    run(p, h, 1, [("extend", [16, 16, 0]), ("draft", [5, 0, 0]), ("extend", [0, 1, 0]), ("release", [1, 0, 0]),
                  ("extend", [0, 0, 40]), ("release", [0, 1, 1])])
    assert sorted(p.free) == list(range(12))


def test_rows_that_would_go_back_to_fewer_full_pages():
    """A full page can be shared: the row that owns it must not fill it again."""
    for lens, parents in (([17, 15], [1, 0]), ([16, 15], [1, 0]), ([20, 12, 20], [2, 1, 0])):
        p, h = O.Owners(len(lens), 4, 12, 16), O.Held(len(lens), 12, 16)
        run(p, h, len(lens), [("extend", lens)])
        before = p.copy()
        assert p.reorder(parents, len(lens))[0] == (0 if lens == [20, 12, 20] else 5)
        if lens != [20, 12, 20]:
            assert np.array_equal(p.owned, before.owned) and np.array_equal(p.table, before.table) and p.lens == before.lens


def test_pages_that_a_row_went_back_from():
    """To the first token of the page it was filling: the page stays the row's and is begun again."""
    p, h = O.Owners(2, 4, 8, 16), O.Held(2, 8, 16)
    seen = run(p, h, 2, [("extend", [20, 16]), ("reorder", [1, 0]), ("draft", [3, 0]), ("extend", [2, 0]), ("extend", [16, 9]),
                         ("draft", [9, 9]), ("reorder", [0, 1]), ("release", [1, 1])])
    assert all(st == 0 for _, st in seen) and sorted(p.free) == list(range(8))
