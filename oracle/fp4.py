"""FP4 page pool, its attention and the page operations in numpy (64 bits), from their definitions."""

from __future__ import annotations

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# nearest, ties to the even code: a magnitude on a border goes up only where the code above is even
BORDERS = (GRID[1:] + GRID[:-1]) / 2


def values(x: np.ndarray) -> np.ndarray:
    """What a pool holds for dense rows [..., D]."""
    x = np.where(np.isnan(x), 0.0, np.asarray(x, np.float64))
    blocks = x.reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    top = np.abs(blocks).max(-1, keepdims=True)
    e = np.full(top.shape, -14.0)
    for k in range(-14, 13):                     # the smallest e with 6 * 2^e >= top, at most 13
        e = np.where(6.0 * 2.0 ** k < top, k + 1.0, e)
    y = np.minimum(np.abs(blocks) / 2.0 ** e, 1e9)
    code = np.zeros(y.shape, int)
    for i, b in enumerate(BORDERS):
        code += (y >= b) if (i + 1) % 2 == 0 else (y > b)
    out = np.sign(blocks) * GRID[code] * 2.0 ** e
    return out.reshape(x.shape)


def _softmax_rows(s):
    m = s.max(-1, keepdims=True) if s.shape[-1] else np.zeros(s.shape[:-1] + (1,))
    m = np.where(np.isfinite(m), m, 0.0)
    p = np.exp(s - m)
    t = p.sum(-1, keepdims=True)
    return np.where(t > 0, p / np.where(t > 0, t, 1.0), 0.0)


def attention(q, k, v, seen, sm_scale):
    """q [R, D], k / v [T, D], seen [R, T] -> (out, spread): spread[r, c] = softmax(..) |v|, the size that rounding
    errors of the probabilities scale with, and reach[r] = max over keys of |sm_scale| sum |q k|."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    s = np.where(seen, sm_scale * (q @ k.T), -np.inf)
    p = _softmax_rows(s)
    reach = (np.abs(q) @ np.abs(k).T * abs(sm_scale) * seen).max(-1, initial=0.0)
    return p @ v, p @ np.abs(v), reach


class Pages:
    """Sequential page operations on numpy copies of refs, table, lengths and a list of page planes [P, ...]."""

    def __init__(self, refs, table, lengths, page_size, planes=()):
        self.refs, self.table, self.lengths = refs.copy(), table.copy(), lengths.copy()
        self.ps, self.planes, self.rejected = page_size, [p.copy() for p in planes], 0

    def held(self, s):
        return min(-(-max(int(self.lengths[s]), 0) // self.ps), self.table.shape[2])

    def grow(self, more):
        S, Ht, W = self.table.shape
        P = len(self.refs)
        refs0 = self.refs.copy()
        free = [p for p in range(P) if refs0[p] <= 0]
        used, full = 0, False
        for s in range(S):
            n, ln = int(more[s]), max(int(self.lengths[s]), 0)
            if n == 0:
                continue
            old = -(-ln // self.ps)
            bad = n < 0 or ln + n > W * self.ps
            if not bad and ln % self.ps:
                bad = any(not 0 <= self.table[s, h, old - 1] < P for h in range(Ht))
            if bad:
                self.rejected += 1
                continue
            new = -(-(ln + n) // self.ps)
            wants = []
            for h in range(Ht):
                if ln % self.ps and refs0[self.table[s, h, old - 1]] > 1:
                    wants.append((h, old - 1, True))
                wants += [(h, w, False) for w in range(old, new)]
            # once a slot does not fit, every later one that gets tokens is refused too
            full = full or used + len(wants) > len(free)
            if full:
                self.rejected += 1
                continue
            for h, w, copy in wants:
                p = free[used]
                used += 1
                if copy:
                    was = self.table[s, h, w]
                    for x in self.planes:
                        x[p] = x[was]
                    self.refs[was] -= 1
                self.refs[p] = 1
                self.table[s, h, w] = p
            self.lengths[s] = ln + n

    def shrink(self, tokens):
        for s, n in enumerate(tokens):
            n, ln = int(n), max(int(self.lengths[s]), 0)
            if n == 0:
                continue
            if n < 0 or n > ln:
                self.rejected += 1
                continue
            a, b = -(-(ln - n) // self.ps), self.held(s)
            for p in self.table[s, :, a:b].ravel():
                if 0 <= p < len(self.refs):
                    self.refs[p] -= 1
            self.table[s, :, a:b] = -1
            self.lengths[s] = ln - n

    def fork(self, src, dst):
        S, P = len(self.lengths), len(self.refs)
        lengths = self.lengths.copy()
        for i, (a, b) in enumerate(zip(src, dst)):
            if not (0 <= a < S and 0 <= b < S) or lengths[b] > 0 or a in dst or b in dst[:i]:
                self.rejected += 1
                continue
            w = self.held(a)
            self.table[b, :, :w] = self.table[a, :, :w]
            for p in self.table[a, :, :w].ravel():
                if 0 <= p < P:
                    self.refs[p] += 1
            self.lengths[b] = lengths[a]

    def free(self, slots):
        for i, s in enumerate(slots):
            if not 0 <= s < len(self.lengths):
                self.rejected += 1
                continue
            if s in slots[:i]:
                continue
            w = self.held(s)
            for p in self.table[s, :, :w].ravel():
                if 0 <= p < len(self.refs):
                    self.refs[p] -= 1
            self.table[s, :, :w] = -1
            self.lengths[s] = 0

    def compact(self):
        n = int((self.refs > 0).sum())
        src = [p for p in range(n, len(self.refs)) if self.refs[p] > 0]
        dst = [p for p in range(n) if self.refs[p] <= 0]
        to = dict(zip(src, dst))
        for a, b in to.items():
            for x in self.planes:
                x[b] = x[a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        for s in range(len(self.lengths)):
            w = self.held(s)
            self.table[s, :, :w] = np.vectorize(lambda p: to.get(p, p), otypes=[np.int32])(self.table[s, :, :w])
        return n
