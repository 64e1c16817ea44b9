"""Plain 64-bit implementation of the paged 4-bit cache, from its definition: the row format, the
step's pages and slots (on Python lists), attention over the values that a cache holds."""

import numpy as np

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def values(x):
    """What the cache holds for rows x [..., 128] (any float array), in float64."""
    x = np.asarray(x, np.float64)
    g = x.reshape(x.shape[:-1] + (4, 32))
    top = np.abs(g).max(-1, keepdims=True)
    fin = np.isfinite(top)
    mant, ex = np.frexp(np.where(fin, top, 0.0))           # top = mant * 2^ex, mant in [1/2, 1)
    e = np.where(mant <= 0.875, ex - 3, ex - 2)            # 7 * 2^-3 = 0.875
    e = np.where(mant == 0, -127, np.maximum(e, -127))
    a = np.where(fin, np.abs(g), 0.0) / np.ldexp(1.0, e)
    code = np.zeros(a.shape, np.int64)
    for c in range(1, 8):                                  # past a midpoint, or on it and c even
        mid = (GRID[c - 1] + GRID[c]) / 2
        code += (a > mid) | ((a == mid) & (c % 2 == 0))
    v = np.copysign(GRID[code], np.where(fin, g, 0.0)) * np.ldexp(1.0, e)
    return np.where(fin, v, np.nan).reshape(x.shape)


def pages(n, page):
    return -(-n // page)


class Plan:
    """The step on lists."""

    def __init__(self, n_seq, page, width, n_pages):
        self.page, self.width, self.n_pages = page, width, n_pages
        self.lens = [0] * n_seq
        self.table = [[] for _ in range(n_seq)]
        self.free = list(range(n_pages - 1, -1, -1))

    def step(self, grow, keep, max_rows):
        """(starts, slots, positions) and 0, or nothing changed and the error bits."""
        n, P = len(self.lens), self.page
        err = 0
        for l, k, g in zip(self.lens, keep, grow):
            if k < 0 or k > l or g < 0 or k + g > self.width * P:
                err |= 8
        none = ([0] * (n + 1), [-1] * max_rows, [-1] * max_rows)
        if err:
            return none, err
        freed = [p for l, k, t in zip(self.lens, keep, self.table) for p in t[pages(k, P):]]
        need = sum(pages(k + g, P) - pages(k, P) for k, g in zip(keep, grow))
        if need > len(self.free) + len(freed):
            err |= 16
        if sum(grow) > max_rows:
            err |= 32
        if err:
            return none, err
        self.free += freed[::-1]
        starts, slots, pos = [0], [], []
        for s in range(n):
            self.table[s] = self.table[s][:pages(keep[s], P)]
            while len(self.table[s]) < pages(keep[s] + grow[s], P):
                self.table[s].append(self.free.pop())
            self.lens[s] = keep[s] + grow[s]
            for r in range(keep[s], self.lens[s]):
                slots.append(self.table[s][r // P] * P + r % P)
                pos.append(r)
            starts.append(len(slots))
        pad = [-1] * (max_rows - len(slots))
        return (starts, slots + pad, pos + pad), 0


def attend(q, k, v, causal, scale):
    """q [m, heads, 128], k and v [n, kv, 128], float64 -> (out, lse, mass, size): mass [m, heads,
    128] is sum w |v| / sum w, size [2, m, heads] the largest over the visible keys of scale * sum
    |q k| and of scale * sum |g k|, g the largest |q| of the value's group of 32."""
    m, heads, _ = q.shape
    n, kv, _ = k.shape
    r = heads // kv
    out = np.zeros((m, heads, 128))
    lse = np.full((m, heads), -np.inf)
    mass = np.zeros((m, heads, 128))
    size = np.zeros((2, m, heads))
    group = np.abs(q).reshape(m, heads, 4, 32).max(-1).repeat(32, -1)
    for h in range(heads):
        if n == 0:
            break
        kk, vv = k[:, h // r], v[:, h // r]
        with np.errstate(invalid="ignore", over="ignore"):
            s = q[:, h] @ kk.T * scale
        for t in range(m):
            see = max(0, min(n, n - m + t + 1)) if causal else n
            if see == 0:
                continue
            x = s[t, :see]
            top = x.max()
            with np.errstate(invalid="ignore"):
                w = np.exp(x - top)
            out[t, h] = w @ vv[:see] / w.sum()
            mass[t, h] = w @ np.abs(vv[:see]) / w.sum()
            lse[t, h] = top + np.log(w.sum())
            size[0, t, h] = scale * (np.abs(q[t, h]) @ np.abs(kk[:see]).T).max()
            size[1, t, h] = scale * (group[t, h] @ np.abs(kk[:see]).T).max()
    return out, lse, mass, size


def attend_tolerance(out, lse, mass, size, n, half_step, split=True):
    """How far a result may be off, by arithmetic.  half_step = eps / 2 of the query's type; split:
    the query goes into the product as three 6-bit parts (tiles of more than 32 rows).

    Logits: 128 products summed in fp32, each sum off by at most 2^-23 (MFMA sums may truncate), of
    at most `size` in all; the product with scale * log2(e), the difference to the reference and
    the power add 4 roundings of numbers up to the logit's size.  So a weight is off by the factor
    1 + d, d <= 2^-23 (132 size + 8).  Weights round to the type: half_step each; their sum is that
    of the rounded ones.  The chain of fp32 sums over n keys has n / 32 steps in a wave, and some 64
    more between waves and workers.  With o = sum w v / sum w, weights off by f each move o by at
    most 2 f sum w |v| / sum w; the result rounds once more.  Weights below 2^-34 of the largest
    may vanish (fp16): n 2^-34 of the mass, which is at least 1 / n of the largest value's.

    The parts of a query have 4 bits: x = (p0 + p1 / 16 + p2 / 512) 2^b with 3.75 2^b < g <= 7.5 2^b
    for the largest |x| = g of 32.  p0 leaves at most 1/4 (half a step of 1/2), which is 4 units of
    p1; p1 leaves at most 1/8 (half a step of 1/4 below 4), which is 4 units of p2; p2 leaves 1/8
    of its unit, 2^(b - 12) <= 2^-12 / 3.75 g.  A logit is off by at most that times size[1].  Its
    384 products add up on the reference's exponent (a logit and KV4_LIFT = 9 in log2, 7), so that
    each of their sums is off by 2^-23 of that, too."""
    d = 2.0 ** -23 * (132 * size[0] + 8 + n / 32 + 64) + n * 2.0 ** -34
    if split:
        d += 2.0 ** -12 / 3.75 * size[1] + 2.0 ** -23 * 384 * (2 * size[0] + 7)
    tol = half_step * np.abs(out) + (2 * half_step + 2 * d)[..., None] * mass + 2.0 ** -24
    return tol, half_step + 2 * d + 2.0 ** -20 * np.maximum(1, np.abs(lse))
