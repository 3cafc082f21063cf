"""The paged MX4 cache, its bookkeeping, rotary positions and attention from
their definitions, in numpy and 64 bits: what the GPU operators are compared
with."""
import numpy as np

import _mx4ref as R


def plan(lengths, new, table, page, free, count, pages, tokens):
    """One request after another."""
    lengths, table, free = list(lengths), table.copy(), free.copy()
    requests, width = table.shape
    n = [max(0, int(v)) for v in new]
    top = min(max(count, 0), pages)

    def held(tokens_):
        return -(-min(max(tokens_, 0), width * page) // page)

    for r in range(requests):
        if new[r] < 0:
            for i in range(held(lengths[r])):
                if top < pages:
                    free[top] = table[r, i]
                    top += 1
    starts, positions, slots, of = [0], np.full(tokens, -1), np.full(tokens, -1), np.full(tokens, -1)
    out, left, needed, unserved, total = [], top, 0, 0, 0
    for r in range(requests):
        past = max(lengths[r], 0)
        total += n[r]
        of[min(tokens, starts[-1]): min(tokens, total)] = r
        wide = past + n[r] > width * page
        need = 0 if new[r] < 0 or wide else -(-(past + n[r]) // page) - held(past)
        needed += need
        if new[r] < 0:
            out.append(0)
        elif wide or total > tokens or (need > 0 and needed > top):
            unserved += 1
            out.append(past)
        else:
            first = held(past)
            for i in range(need):
                left -= 1
                table[r, first + i] = free[left]
            for i in range(n[r]):
                positions[starts[-1] + i] = past + i
                number = table[r, (past + i) // page]
                slots[starts[-1] + i] = number * page + (past + i) % page if 0 <= number < pages else -1
            out.append(past + n[r])
        starts.append(min(total, tokens))
    return {"starts": np.array(starts), "lengths": np.array(out), "table": table, "free": free[:top], "left": left,
            "unserved": unserved, "positions": positions, "slots": slots, "requests": of}


def turned(x, positions, frequencies, factor=1.0, interleaved=False, back=False):
    """x: tokens x heads x dim; rows of positions below zero as they are."""
    x = np.asarray(x, np.float64)
    half = len(frequencies)
    t = np.asarray(positions, np.float64)[:, None, None] * np.asarray(frequencies, np.float64)
    c, s = np.cos(t) * factor, np.sin(t) * (-factor if back else factor)
    a, b = (x[..., 0: 2 * half: 2], x[..., 1: 2 * half: 2]) if interleaved else (x[..., :half], x[..., half: 2 * half])
    y = x.copy()
    p, q = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0: 2 * half: 2], y[..., 1: 2 * half: 2] = p, q
    else:
        y[..., :half], y[..., half: 2 * half] = p, q
    return np.where((np.asarray(positions) < 0)[:, None, None], x, y)


class Cache:
    """The bytes of a cache: pages x heads x a head's bytes."""

    def __init__(self, pages, page, heads, dim):
        self.pages, self.page, self.heads, self.dim = pages, page, heads, dim
        self.blocks = -(-dim // 32)
        self.row, self.decoded = 16 * self.blocks, None
        self.bytes = np.zeros((pages, heads, 34 * self.blocks * page), np.uint8)

    def codes(self, number, h, which, t):
        at = (which * self.page + t) * self.row
        return self.bytes[number, h, at: at + self.row]

    def scale_index(self, which, t):
        begin = 2 * self.page * self.row + which * self.page * self.blocks + t // 16 * 16 * self.blocks
        return begin + 4 * (t % 4 * self.blocks + np.arange(self.blocks)) + t % 16 // 4

    def put(self, slot, k, v):
        """k, v: heads x dim, in 64 bits."""
        self.decoded = None
        if not 0 <= slot < self.pages * self.page:
            return
        for h in range(self.heads):
            for which, x in enumerate((k[h], v[h])):
                codes, scales = R.packed(x)
                self.codes(slot // self.page, h, which, slot % self.page)[:] = codes[: self.row]
                self.bytes[slot // self.page, h, self.scale_index(which, slot % self.page)] = scales[: self.blocks]

    def get(self, slot, h, which):
        return self.values(which)[slot, h]

    def values(self, which):
        """All of the keys or values, slots x heads x dim."""
        if self.decoded is None:
            t = np.arange(self.page)
            at = np.stack([self.scale_index(0, i) for i in t])  # of the page's tokens
            self.decoded = []
            for w in (0, 1):
                c = self.bytes[:, :, w * self.page * self.row: (w + 1) * self.page * self.row]
                c = c.reshape(self.pages, self.heads, self.page, self.row)
                code = np.stack((c & 15, c >> 4), -1).reshape(*c.shape[:3], -1)
                x = R.decode(code, self.bytes[:, :, at + w * self.page * self.blocks], self.dim)
                self.decoded.append(x.transpose(0, 2, 1, 3).reshape(-1, self.heads, self.dim))
        return self.decoded[which]


def attention(cache, row, length, q, scale, causal=True, window=0, most=None):
    """One request: q (n x query heads x dim).  out, lse, and for each (query,
    head) what its error is measured by: (sum of p |v|, the largest sum of
    |scale q k|, the spread of the scores, sum of |v|)."""
    n, heads, dim = q.shape
    group = heads // cache.heads
    seen_pages = [0 <= row[j // cache.page] < cache.pages for j in range(length)]
    out, lse = np.zeros((n, heads, dim)), np.full((n, heads), -np.inf)
    of = np.zeros((n, heads, dim)), np.zeros((n, heads)), np.zeros((n, heads)), np.zeros((n, heads, dim))
    for h in range(cache.heads):
        slots = np.array([int(row[j // cache.page]) * cache.page + j % cache.page if seen_pages[j] else 0 for j in range(length)], int)
        k, v = cache.values(0)[slots, h], cache.values(1)[slots, h]
        for i in range(n):
            at = length - n + i
            see = [seen_pages[j] and (not causal or (j <= at and (window == 0 or j > at - window))) for j in range(length)]
            see = np.array(see, bool).reshape(length)
            if not see.any():
                continue
            for head in range(h * group, (h + 1) * group):
                with np.errstate(invalid="ignore"):
                    score = k[see] @ q[i, head].astype(np.float64) * scale
                    top = score.max()
                    p = np.exp(score - top)
                    out[i, head] = p @ v[see] / p.sum()
                    lse[i, head] = top + np.log(p.sum())
                    of[0][i, head] = p @ np.abs(v[see]) / p.sum()
                    of[1][i, head] = np.abs(scale) * (np.abs(k[see]) @ np.abs(q[i, head])).max()
                    of[2][i, head] = np.abs(score).max() + (top - score.min())
                    of[3][i, head] = np.abs(v[see]).sum(0)
    return out, lse, of


def attention_bound(of, keys, dim, depth, rounding):
    """How far (out, lse) may be off.  depth: BF16 pieces of queries and weights.
    A score is a sum of depth * dim products (exact ones), off by 2^-23 of the
    magnitudes for each addition, and then a few roundings of itself and of its
    distance from the reference; a weight is off by as much relatively, by 2^-21
    in exp2, and by 2^-8 depth where it goes into the products.  Sums over the
    keys: 2^-23 for each addition and piece, and for the joins.

    Weights, and pieces of weights, below 2^-126 may be zero: up to three of those
    for each key, over a sum of at least 2^-8 (the reference lies up to 8 below the
    largest score): 3 * 2^-126 * 2^8 < 2^-116 of every |v|."""
    weighed, products, spread, magnitudes = of
    score = depth * dim * 2.0**-23 * products + 2.0**-22 * spread
    weight = score + 2.0**-21
    adds = (depth * keys + 64) * 2.0**-23
    out = (2 * weight + 2.0**(-8 * depth) + 2 * adds)[..., None] * weighed + 2.0**-116 * magnitudes
    return out, weight + adds + 2.0**-22 * spread, rounding
