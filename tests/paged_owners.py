"""Who owns a page of the paged cache: a plain implementation of its plans, and a check of it that knows nothing of its rules.

An entry of `owned` counts as a page of its row
  - where it is an id and its place lies below the pages that the row's tokens reach (j < ceil(lens / page)): what lies past
    them is left of a step that was dropped, and that page is on the stack;
  - where it is -2 - id: a page that its row began and then went back from, by a reordering, to the place's first token. The
    row begins it again when it comes back to the place.
"""
import numpy as np


class Owners:
    def __init__(self, n_requests, max_pages, n_pages, page):
        self.page, self.n_pages, self.max_pages = page, n_pages, max_pages
        self.lens = [0] * n_requests
        self.table = np.full((n_requests, max_pages), -1, np.int32)
        self.owned = self.table.copy()
        self.stack, self.height = list(range(n_pages - 1, -1, -1)), n_pages

    def copy(self):
        new = object.__new__(Owners)
        new.__dict__ = {k: v.copy() if hasattr(v, "copy") else v for k, v in self.__dict__.items()}
        return new

    @property
    def free(self):
        return self.stack[:self.height]

    def pages(self, tokens):
        return -(-tokens // self.page)

    def page_of(self, r, j, used=None):
        """The page that row r owns at place j, or -1."""
        v = int(self.owned[r, j])
        return -2 - v if v <= -2 else v if j < (self.pages(self.lens[r]) if used is None else used) else -1

    def extend(self, n_new, drop=False):
        """(status, slots, positions, requests). drop: lengths and height stay, as if the caller had kept the outputs apart."""
        lens, height = list(self.lens), self.height
        ends = [a + n for a, n in zip(lens, n_new)]
        if any(self.pages(e) > self.max_pages for e in ends):
            return 2, [], [], []
        kept = [self.page_of(r, self.pages(a)) if self.pages(e) > self.pages(a) else -1 for r, (a, e) in enumerate(zip(lens, ends))]
        need = sum(self.pages(e) - self.pages(a) - (k >= 0) for a, e, k in zip(lens, ends, kept))
        if need > height:
            return 1, [], [], []
        slots, positions, requests = [], [], []
        for r, (a, e) in enumerate(zip(lens, ends)):
            for j in range(self.pages(a), self.pages(e)):
                if j == self.pages(a) and kept[r] >= 0:
                    self.table[r, j] = kept[r]
                else:
                    height -= 1
                    self.table[r, j] = self.owned[r, j] = self.stack[height]
            for pos in range(a, e):
                slots.append(int(self.table[r, pos // self.page]) * self.page + pos % self.page)
                positions.append(pos)
                requests.append(r)
        if not drop:
            self.lens, self.height = ends, height
        return 0, slots, positions, requests

    def release(self, ended):
        for r, e in enumerate(ended):
            if e:
                for j in range(self.max_pages):
                    page = self.page_of(r, j)
                    if page >= 0:
                        self.stack[self.height] = page
                        self.height += 1
                self.owned[r] = self.table[r] = -1
                self.lens[r] = 0

    def reorder(self, parent, width):
        """(status, [(from page, to page, rows)] of the open pages that move)."""
        rows = [(r // width * width + q if 0 <= q < width else r) for r, q in enumerate(parent)]
        old, new = list(self.lens), [self.lens[p] for p in rows]
        if any(a // self.page > b // self.page for a, b in zip(old, new)):
            return 5, []
        need = [r for r, n in enumerate(new) if n % self.page and self.page_of(r, n // self.page) < 0]
        if len(need) > self.height:
            return 1, []
        sources = [self.page_of(p, n // self.page) if n % self.page else -1 for p, n in zip(rows, new)]
        for r in range(len(rows)):
            a, b = self.pages(old[r]), self.pages(new[r])
            for j in range(a, b):  # (left of dropped steps: not to be counted now that the row reaches further)
                if self.owned[r, j] >= 0:
                    self.owned[r, j] = -1
            if b < a and self.owned[r, b] >= 0:
                self.owned[r, b] = -2 - self.owned[r, b]
            if new[r] % self.page and self.owned[r, b - 1] <= -2:
                self.owned[r, b - 1] = -2 - self.owned[r, b - 1]
        for r in need:
            self.height -= 1
            self.owned[r, new[r] // self.page] = self.stack[self.height]
        table, moves = np.full_like(self.table, -1), []
        self.lens = new
        for r, p in enumerate(rows):
            j = new[r] // self.page
            table[r, :j] = self.table[p, :j]
            if new[r] % self.page:
                table[r, j] = self.page_of(r, j)
                if p != r:
                    moves.append((sources[r], int(table[r, j]), new[r] % self.page))
        self.table = table
        return 0, moves


class Held:
    """What each row should hold (its tokens, by a number of their own) and what each place of the cache does hold."""

    def __init__(self, n_requests, n_pages, page):
        self.page, self.cells = page, np.full((n_pages, page), -1, np.int64)
        self.rows, self.next = [[] for _ in range(n_requests)], 0

    def write(self, slots, requests, keep=True):
        for s, r in zip(slots, requests):
            self.cells[s // self.page, s % self.page] = self.next
            if keep:
                self.rows[r].append(self.next)
            self.next += 1

    def reorder(self, parent, width, moves):
        rows = [(r // width * width + q if 0 <= q < width else r) for r, q in enumerate(parent)]
        self.rows = [list(self.rows[p]) for p in rows]
        old = self.cells.copy()
        for src, dst, n in moves:
            self.cells[dst, :n] = old[src, :n]

    def release(self, ended):
        self.rows = [[] if e else x for x, e in zip(self.rows, ended)]


def check(pages, held, width):
    """Every row reads what it should; no page is both free and a row's, none has two owners, none is lost; every page in use
    is owned by a row of its group, and one that is still being filled is read by its owner alone."""
    page, n = pages.page, pages.n_pages
    free = [int(x) for x in pages.free]
    assert len(set(free)) == len(free) and all(0 <= x < n for x in free)
    owner = {}
    for r in range(len(pages.lens)):
        for j in range(pages.max_pages):
            x = pages.page_of(r, j)
            if x >= 0:
                assert x not in owner, f"page {x} has the owners {owner[x]} and {(r, j)}"
                owner[x] = (r, j)
    assert not set(free) & set(owner), "a page in use is on the stack"
    assert len(free) + len(owner) == n, "pages are lost"
    readers = {}
    for r, length in enumerate(pages.lens):
        assert len(held.rows[r]) == length
        for t in range(length):
            x = int(pages.table[r, t // page])
            assert x in owner and owner[x][0] // width == r // width
            assert held.cells[x, t % page] == held.rows[r][t], f"row {r}, token {t}"
            readers.setdefault(x, set()).add(r)
    for r, length in enumerate(pages.lens):
        if length % page:
            x = int(pages.table[r, length // page])
            assert owner[x] == (r, length // page) and readers[x] == {r}


def steps(rng, groups, width, page, max_pages, n_steps, unequal, drafts=True):
    """A random sequence of calls: ("extend", counts), ("draft", counts), ("reorder", parents), ("release", flags).

    A group starts with a prompt in its first row, handed to the others; then its rows get equally many tokens, or with
    `unequal` none for rows that count as finished.
    """
    b = groups * width
    started, finished = np.zeros(groups, bool), np.zeros((groups, width), bool)
    for _ in range(n_steps):
        what = rng.random()
        if what < 0.1:
            ended = rng.random(groups) < 0.4
            started &= ~ended
            finished &= ~ended[:, None]
            yield "release", np.repeat(ended, width).astype(int).tolist()
        n = np.zeros((groups, width), int)
        for g in range(groups):
            if started[g]:
                n[g] = 1 if rng.random() < 0.6 else rng.integers(1, 2 * page)
                if rng.random() < 0.2:
                    n[g] = 0
                n[g][finished[g]] = 0
            else:
                n[g, 0] = rng.integers(1, 3 * page)
        if drafts and what < 0.5:  # drafted, dropped, and some of it taken up
            draft = n + rng.integers(0, page + 2, n.shape)
            yield "draft", draft.reshape(-1).tolist()
            if rng.random() < 0.5:
                yield "draft", (draft + rng.integers(-1, 2, n.shape)).clip(0).reshape(-1).tolist()
        yield "extend", n.reshape(-1).tolist()
        if what > 0.25:
            parent = rng.integers(0, width, (groups, width))
            for g in range(groups):
                if not started[g]:
                    parent[g] = 0
                elif rng.random() < 0.3:
                    parent[g] = np.arange(width)
            yield "reorder", parent.reshape(-1).tolist()
            for g in range(groups):
                started[g] = True
                finished[g] = finished[g][parent[g]]
                if unequal:
                    finished[g] |= rng.random(width) < 0.1
        else:  # (a group goes on only from a reordering that handed its prompt on)
            ended = ~started
            if ended.any():
                yield "release", np.repeat(ended, width).astype(int).tolist()
