"""Plain implementations, in numpy and 64 bits, of the paged cache's operators: what the GPU tests compare with."""
import math

import numpy as np


class Pages:
    """A batch's requests and their pages, as jk_paged describes them."""

    def __init__(self, n_requests, max_pages, n_pages, page):
        self.page, self.n_pages, self.max_pages = page, n_pages, max_pages
        self.lens = [0] * n_requests
        self.table = np.full((n_requests, max_pages), -1, np.int32)
        self.owned = self.table.copy()
        self.free = list(range(n_pages - 1, -1, -1))

    def pages(self, tokens):
        return -(-tokens // self.page)

    def extend(self, n_new, max_tokens):
        """(status, q_start, slots, positions, requests); nothing changes where status is not 0."""
        b = len(self.lens)
        none = ([0] * (b + 1), [-1] * max_tokens, [-1] * max_tokens, [-1] * max_tokens)
        if any(n < 0 or ln < 0 or self.pages(ln) > self.max_pages for n, ln in zip(n_new, self.lens)):
            return (3,) + none
        if any(self.pages(n + ln) > self.max_pages for n, ln in zip(n_new, self.lens)) or sum(n_new) > max_tokens:
            return (2,) + none
        if sum(self.pages(n + ln) - self.pages(ln) for n, ln in zip(n_new, self.lens)) > len(self.free):
            return (1,) + none
        q_start, slots, positions, requests = [0], [], [], []
        for r, n in enumerate(n_new):
            for i in range(n):
                pos = self.lens[r]
                if pos % self.page == 0:
                    self.table[r, pos // self.page] = self.owned[r, pos // self.page] = self.free.pop()
                slots.append(int(self.table[r, pos // self.page]) * self.page + pos % self.page)
                positions.append(pos)
                requests.append(r)
                self.lens[r] += 1
            q_start.append(len(slots))
        pad = [-1] * (max_tokens - len(slots))
        return 0, q_start, slots + pad, positions + pad, requests + pad

    def release(self, ended):
        for r, e in enumerate(ended):
            if e:
                self.free += [int(x) for x in self.owned[r] if x >= 0]
                self.owned[r] = self.table[r] = -1
                self.lens[r] = 0

    def reorder(self, parent, width):
        """(status, [(from page, to page, rows)] of the open pages that move)."""
        rows = [(r // width * width + q if 0 <= q < width else r) for r, q in enumerate(parent)]
        lens = [self.lens[p] for p in rows]
        need = []
        for r, p in enumerate(rows):
            j = lens[r] // self.page
            if lens[r] % self.page:
                if self.owned[p, j] < 0 or self.owned[p, j] != self.table[p, j]:
                    return 4, []
                if self.owned[r, j] < 0:
                    need.append((r, j))
        if len(need) > len(self.free):
            return 1, []
        for r, j in need:
            self.owned[r, j] = self.free.pop()
        table, moves = np.full_like(self.table, -1), []
        for r, p in enumerate(rows):
            j = lens[r] // self.page
            table[r, :j] = self.table[p, :j]
            if lens[r] % self.page:
                table[r, j] = self.owned[r, j]
                if p != r:
                    moves.append((int(self.owned[p, j]), int(self.owned[r, j]), lens[r] % self.page))
        self.lens, self.table = lens, table
        return 0, moves


def append(codes, scale, x, slots):
    """Stores x [t][heads][hd] in codes [pages][heads][page][hd] and scale [pages][heads], in place, in f32 as defined."""
    page, t = codes.shape[2], 0
    x = np.where(np.isfinite(x), x, 0).astype(np.float32)
    while t < len(slots):
        if not 0 <= slots[t] < codes.shape[0] * page:
            t += 1
            continue
        p, e = slots[t] // page, t + 1
        while e < len(slots) and slots[e] // page == p and slots[e] > slots[e - 1]:
            e += 1
        rows = [s % page for s in slots[t:e]]
        for h in range(codes.shape[1]):
            top = np.float32(np.abs(x[t:e, h]).max())
            old = np.float32(0) if rows[0] == 0 else scale[p, h]
            if not (np.isfinite(old) and old > 0):
                old = np.float32(0)
            d = max(old, np.float32(0) if top < 2.0 ** -119 else top / np.float32(127))
            if rows[0] and d != old:
                codes[p, h, :rows[0]] = np.rint(codes[p, h, :rows[0]].astype(np.float32) * (old / d)).astype(np.int8)
            inv = np.float32(1) / d if d > 0 else np.float32(0)
            codes[p, h, rows] = np.clip(np.rint(x[t:e, h] * inv), -127, 127).astype(np.int8)
            scale[p, h] = d
        t = e


def attention(q, codes_k, codes_v, scale_k, scale_v, q_start, lens, table, scale, window, unit):
    """(out, bound): the outputs in 64 bits, and how far a computed one may be from them.

    unit: the roundings to dtype (2^-24 for f32 ..) of probabilities and of the output. The bound of a row with largest
    visible |v| = V and n keys: the scores are sums of hd f32 products of codes with queries held to 2^-21 of their row's
    largest value, off by at most e_s = scale * hd * max|q| * max|k| * (hd 2^-24 + 2^-21) + 2^-23 max|s| (the product with
    log2(e) and the scales); each p is then off by e_s + 2^-21 of itself (exponential, subtraction of the maximum), the weighted sum by twice
    that (p above and below) plus n 2^-24 of V (its additions), and the rounding of the weights adds w V, of the output u |o|.
    """
    w, u = unit
    t, heads, hd = q.shape
    page, kv = codes_k.shape[2], codes_k.shape[1]
    grp = heads // kv
    out = np.full(q.shape, np.nan)
    bound = np.zeros(q.shape)
    for r, ln in enumerate(lens):
        first, last = q_start[r], q_start[r + 1]
        for i in range(last - first):
            pos = ln - (last - first) + i
            js = [j for j in range(max(0, pos - window + 1 if window else 0), pos + 1)
                  if j < ln and 0 <= table[r, j // page] < codes_k.shape[0]]
            for e in range(heads):
                h = e // grp
                if not js:
                    out[first + i, e] = 0
                    continue
                ps, rows = table[r, np.array(js) // page], np.array(js) % page
                k = codes_k[ps, h, rows].astype(np.float64) * scale_k[ps, h, None].astype(np.float64)
                v = codes_v[ps, h, rows].astype(np.float64) * scale_v[ps, h, None].astype(np.float64)
                x = q[first + i, e].astype(np.float64)
                s = k @ x * scale
                p = np.exp(s - s.max())
                o = p @ v / p.sum()
                out[first + i, e] = o
                big = abs(scale) * hd * np.abs(x).max() * np.abs(k).max()
                e_s = big * (hd * 2.0 ** -24 + 2.0 ** -21) + np.abs(s).max() * 2.0 ** -23
                bound[first + i, e] = np.abs(v).max() * (2 * (e_s + 2.0 ** -21) + len(js) * 2.0 ** -24 + w) + u * np.abs(o)
    return out, bound


def beam(logits, scores, done, eos):
    """(totals, parents, tokens) of a group: logits [width][vocab], in 64 bits, in the defined order."""
    width = len(scores)
    cand = []
    for b in range(width):
        if done is not None and done[b]:
            cand.append((-scores[b], b, 0.0, eos))
            continue
        x = np.where(np.isnan(logits[b]), -np.inf, logits[b]).astype(np.float64)
        m = x.max()
        with np.errstate(invalid="ignore"):
            lse = math.log(np.exp(x - m).sum()) if np.isfinite(m) else math.nan
            total = scores[b] + (x - m - lse)
        total = np.where(np.isnan(total), -np.inf, total)
        order = np.lexsort((np.arange(len(x)), -x))[:width]
        cand += [(-total[t], b, -x[t], int(t)) for t in order]
    cand.sort(key=lambda c: c[:2])  # (stable: within a row the order by logit and token stays)
    best = cand[:width]
    return [-c[0] for c in best], [c[1] for c in best], [c[3] for c in best]
