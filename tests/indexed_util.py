"""Definitions in 64 bits of the row and page operators, for their tests: the embedding lookup and gradient with the
error bounds that follow from their arithmetic, and the bookkeeping of a page cache, one request after another."""
import numpy as np
import torch

FLOATS = (torch.float32, torch.float16, torch.bfloat16)
U32 = 2.0 ** -24  # half a step of fp32, relative


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def floor_of(dtype):
    """Half the distance of two neighbours below the smallest normal number: what a result there may be off by."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def bound_of_rounding(exact, before, dtype):
    """How far a result may be from `exact` whose value in fp32 is off by `before` (absolute) before it is rounded."""
    return before + half_step(dtype) * (exact.abs() + before) + floor_of(dtype)


def lookup(table, ids, first, scale):
    """The exact result and the bound of a lookup: scale is rounded to fp32, the product is rounded to fp32."""
    t = table.double().cpu()
    rows = ids.reshape(-1).cpu().to(torch.int64)
    # (compared as Python would: ids near the ends of int64 must not wrap)
    inside = (rows >= first) & (rows < first + t.shape[0])
    at = torch.where(inside, rows - first * inside, torch.zeros_like(rows))
    out = torch.where(inside[:, None], t[at] * scale, torch.zeros((), dtype=torch.float64))
    return out, out.abs() * (2 * U32 + U32 * U32)


def grad(grads, ids, rows, first, scale, padding, old=None):
    """The exact result and the bound of what precedes its rounding: a sum of m terms in any order is off by at most
    (m - 1) U32 / (1 - (m - 1) U32) times the sum of magnitudes; scale and the product with it add two roundings, the
    sum with what was there before one."""
    width = grads[0].shape[1]
    total = torch.zeros((rows, width), dtype=torch.float64)
    size = torch.zeros((rows, width), dtype=torch.float64)
    count = torch.zeros(rows, dtype=torch.float64)
    for g, i in zip(grads, ids):
        i = i.reshape(-1).cpu().to(torch.int64)
        ok = (i >= first) & (i < first + rows)
        if padding is not None:
            ok &= i != padding
        at = (i[ok] - first)
        total.index_add_(0, at, g.double().cpu()[ok])
        size.index_add_(0, at, g.double().cpu()[ok].abs())
        count.index_add_(0, at, torch.ones(at.numel(), dtype=torch.float64))
    err = abs(scale) * size * (count[:, None] + 2) * U32 * 1.001
    total = total * scale
    if old is not None:
        named = (count > 0)[:, None]
        total = torch.where(named, total + old.double().cpu(), old.double().cpu())
        err = torch.where(named, err + U32 * (total.abs() + err), torch.zeros_like(err))
    return total, err, count


def check(got, exact, before, what=""):
    off = (got.double().cpu() - exact).abs()
    bound = bound_of_rounding(exact, before, got.dtype)
    assert bool(torch.isfinite(bound).all()), f"{what}: the definition and its bound are not finite"
    bad = ~(off <= bound)  # (NaN is within no bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} values too far off, the worst by " \
                          f"{float((off / bound).max()):.3g} bounds, first at {bad.nonzero()[0].tolist()}"


class Books:
    """Bookkeeping and contents of a page cache, by the definition: one request at a time, on the host."""

    def __init__(self, contents, page_tokens, sequences, per_seq):
        self.contents = [np.array(c) for c in contents]  # per pool: [pages, bytes]
        self.pages, self.pt = self.contents[0].shape[0], page_tokens
        self.refs = np.zeros(self.pages, np.int64)
        self.tables = np.full((sequences, per_seq), -1, np.int64)
        self.lengths = np.zeros(sequences, np.int64)
        self.refused = self.moved = self.live = 0

    def used(self, q):
        return -(-int(self.lengths[q]) // self.pt)

    def _sound(self, q):
        return 0 <= q < len(self.lengths)

    def extend(self, seqs, lengths):
        # the free pages are those before the call, handed out in order; a request that asks for more than are left
        # is refused, and so is every later one that needs any: its place in the order is behind the one refused
        free, given, seen, self.refused = np.flatnonzero(self.refs == 0), 0, set(), 0
        for q, n in zip(seqs, lengths):
            ok = self._sound(q) and q not in seen and self.lengths[q] <= n <= self.tables.shape[1] * self.pt
            if self._sound(q):
                seen.add(q)
            if not ok:
                self.refused += 1
                continue
            have, want = self.used(q), -(-int(n) // self.pt)
            first, given = given, given + want - have
            if want > have and given > len(free):
                self.refused += 1
                continue
            self.tables[q, have:want] = free[first:given]
            self.refs[free[first:given]] = 1
            self.lengths[q] = n

    def fork(self, parents, children):
        free, given, seen, self.refused = np.flatnonzero(self.refs == 0), 0, set(), 0
        before = self.lengths.copy()
        for p, c in zip(parents, children):
            ok = self._sound(c) and c not in seen and self._sound(p) and before[c] == 0
            if self._sound(c):
                seen.add(c)
            if not ok:
                self.refused += 1
                continue
            whole, rest = divmod(int(before[p]), self.pt)
            if rest:
                given += 1
                if given > len(free):
                    self.refused += 1
                    continue
                new, old = free[given - 1], self.tables[p, whole]
                for pool in self.contents:
                    pool[new] = pool[old]
                self.tables[c, whole], self.refs[new] = new, 1
            self.tables[c, :whole] = self.tables[p, :whole]
            np.add.at(self.refs, self.tables[p, :whole], 1)
            self.lengths[c] = before[p]

    def free(self, seqs):
        for q in seqs:
            if self._sound(q):
                np.add.at(self.refs, self.tables[q, :self.used(q)], -1)
                self.tables[q], self.lengths[q] = -1, 0

    def compact(self):
        alive = np.flatnonzero(self.refs > 0)
        self.live = len(alive)
        holes = np.flatnonzero(self.refs[:self.live] == 0)
        movers = alive[alive >= self.live]
        self.moved = len(movers)
        for src, dst in zip(movers, holes):
            for pool in self.contents:
                pool[dst] = pool[src]
            self.tables[self.tables == src] = dst
            self.refs[dst], self.refs[src] = self.refs[src], 0
