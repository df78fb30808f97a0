"""The 4-bit K/V cache from its definitions, in numpy and 64 bits (no code of the library)."""

import math

import numpy as np

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def encode(x):
    """x [..., D] float64 -> (codes uint8 [..., D / 2], scales uint8 [..., D / 32])."""
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    bad = ~np.isfinite(g).all(-1)
    a = np.where(bad[..., None], 0.0, np.abs(g))
    part, e = np.frexp(a.max(-1))
    # exponent of the largest magnitude rounded to two significant bits, half up
    e = np.where(a.max(-1) > 0, e - 1 + (part >= 0.875), -2000)
    e = np.clip(e - 2, -125, 125)
    y = np.ldexp(a, -e[..., None])
    off = np.abs(y[..., None] - GRID)
    near = off.min(-1, keepdims=True)
    tied = off == near  # of two equally near codes the even one; past 6 only 6 is near
    even = np.where(tied & (np.arange(8) % 2 == 0), np.arange(8), -1).max(-1)
    code = np.where(even >= 0, even, tied.argmax(-1))
    code = code + 8 * np.signbit(g)
    code = np.where(bad[..., None], 0, code).reshape(*x.shape[:-1], x.shape[-1] // 2, 2).astype(np.uint8)
    return code[..., 0] | (code[..., 1] << 4), np.where(bad, 255, e + 127).astype(np.uint8)


def decode(codes, scales):
    """The values, float64 [..., D]."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], codes.shape[-1] * 2)
    v = np.where(c >= 8, -1.0, 1.0) * GRID[c & 7]
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(np.int64) - 127))
    return (v.reshape(*scales.shape, 32) * s[..., None]).reshape(v.shape)


def parts(page, size, d):
    """A head's part of pages [..., bytes] -> K codes, V codes, K scales, V scales (views)."""
    n, out = 0, []
    for width in (d // 2, d // 2, d // 32, d // 32):
        out.append(page[..., n:n + size * width].reshape(*page.shape[:-1], size, width))
        n += size * width
    assert n == page.shape[-1]
    return out


def tokens(pages, row, n, size, d):
    """K, V float64 [Hkv, n, D] of the first n tokens of a table row, NaN where it names no page."""
    h = pages.shape[1]
    k, v = np.full((h, n, d), np.nan), np.full((h, n, d), np.nan)
    for j in range(0, n, size):
        p = int(row[j // size])
        if 0 <= p < len(pages):
            kc, vc, ks, vs = parts(pages[p], size, d)
            m = min(size, n - j)
            k[:, j:j + m], v[:, j:j + m] = decode(kc, ks)[:, :m], decode(vc, vs)[:, :m]
    return k, v


def attend(q, k, v, count, causal, scale):
    """q [Hq, T, D], k, v [Hkv, N, D] -> out, lse, and `spread` = softmax |v| and `logit` = the largest
    sum |q k| * scale of a row, which error bounds need."""
    hq, t, d = q.shape
    g, n = hq // k.shape[0], k.shape[1]
    out, lse = np.zeros((hq, t, d)), np.full((hq, t), -math.inf)
    spread, logit = np.zeros((hq, t, d)), np.zeros((hq, t))
    for h in range(hq):
        for i in range(count):
            seen = min(max(n - count + i + 1, 0), n) if causal else n
            if seen == 0:
                continue
            s = (k[h // g, :seen] @ q[h, i]) * scale
            top = s.max()
            p = np.exp(s - top)
            lse[h, i] = top + math.log(p.sum()) if not np.isnan(top) else np.nan
            out[h, i] = (p / p.sum()) @ v[h // g, :seen]
            spread[h, i] = (p / p.sum()) @ np.abs(v[h // g, :seen])
            logit[h, i] = (np.abs(k[h // g, :seen]) @ np.abs(q[h, i])).max() * scale
    return out, lse, spread, logit


class Pages:
    """The page calls, one after another on lists."""

    def __init__(self, num_pages, sequences, wide, size):
        self.table = np.full((sequences, wide), -1, np.int32)
        self.lengths = np.zeros(sequences, np.int32)
        self.refs = np.zeros(num_pages, np.int32)
        self.size, self.wide = size, wide

    def _pages(self, n):
        return -(-int(n) // self.size)

    def _free(self):
        return [p for p in range(len(self.refs)) if self.refs[p] == 0]

    def reserve(self, ids, counts):
        """(status, starts)"""
        n, fail = len(ids), lambda code: (code, [-1] * len(ids))
        if any(i < 0 or i >= len(self.lengths) for i in ids):
            return fail(1)
        if len(set(ids)) < n:
            return fail(2)
        if any(c < 0 for c in counts):
            return fail(3)
        if any(self.lengths[i] + c > self.wide * self.size for i, c in zip(ids, counts)):
            return fail(4)
        need = [self._pages(self.lengths[i] + c) - self._pages(self.lengths[i]) for i, c in zip(ids, counts)]
        free = self._free()
        if sum(need) > len(free):
            return fail(5)
        starts = []
        for i, c, k in zip(ids, counts, need):
            at = self._pages(self.lengths[i])
            for j in range(k):
                p = free.pop(0)
                self.table[i, at + j], self.refs[p] = p, 1
            starts.append(int(self.lengths[i]))
            self.lengths[i] += c
        return 0, starts

    def free(self, ids, firsts=None, counts=None):
        if any(i < 0 or i >= len(self.lengths) for i in ids):
            return 1
        if len(set(ids)) < len(ids):
            return 2
        todo = []
        for x, i in enumerate(ids):
            held = self._pages(self.lengths[i])
            first = firsts[x] if firsts is not None else 0
            count = counts[x] if counts is not None and counts[x] >= 0 else held - first
            if first < 0 or count < 0 or first + count > held:
                return 3
            todo.append((i, first, count, held))
        for i, first, count, held in todo:
            row = self.table[i, :held].tolist()
            for p in row[first:first + count]:
                self.refs[p] -= 1
            lost = sum(min(self.size, int(self.lengths[i]) - j * self.size) for j in range(first, first + count))
            row = row[:first] + row[first + count:]
            self.table[i] = row + [-1] * (self.wide - len(row))
            self.lengths[i] -= lost
        return 0

    def fork(self, src, dst, share):
        """(status, [(from, to), ..] page copies)"""
        if any(i < 0 or i >= len(self.lengths) for i in src + dst):
            return 1, []
        if len(set(dst)) < len(dst) or set(src) & set(dst):
            return 2, []
        if any(self.lengths[i] for i in dst):
            return 6, []
        own = [[j for j in range(self._pages(self.lengths[s])) if not share or (j + 1) * self.size > self.lengths[s]]
               for s in src]
        free = self._free()
        if sum(map(len, own)) > len(free):
            return 5, []
        moves = []
        for s, d, mine in zip(src, dst, own):
            self.lengths[d] = self.lengths[s]
            for j in range(self._pages(self.lengths[s])):
                p = int(self.table[s, j])
                if j in mine:
                    moves.append((p, free.pop(0)))
                    p = moves[-1][1]
                self.table[d, j] = p
                self.refs[p] += 1
        return 0, moves

    def compact(self):
        """(live, [(from, to), ..])"""
        live = int((self.refs > 0).sum())
        moves = list(zip([p for p in range(live, len(self.refs)) if self.refs[p]], [p for p in range(live) if not self.refs[p]]))
        to = dict(moves)
        for a, b in moves:
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = np.array([[to.get(int(p), int(p)) for p in row] for row in self.table], np.int32)
        return live, moves
