"""Plain 64-bit implementation of the verification of drafted blocks, from its definition."""

import numpy as np


def distribution(row, temp):
    """softmax(row / temp) in float64, all weight on the first largest below 1e-5; None for a row
    that holds a NaN or +infinity, or nothing above -infinity."""
    x = np.asarray(row, np.float64)
    if np.isnan(x).any() or np.isposinf(x).any() or np.isneginf(x).all():
        return None
    if not temp >= 1e-5:
        p = np.zeros_like(x)
        p[int(np.argmax(x))] = 1.0
        return p
    w = np.exp((x - x.max()) / np.float64(temp))
    return w / w.sum()


def draw(weights, u):
    """The first place whose running sum exceeds u times the whole; the last with any weight if
    rounding leaves none."""
    sums = np.cumsum(weights)
    hit = np.nonzero(sums > np.float64(u) * sums[-1])[0]
    return int(hit[0]) if len(hit) else int(np.nonzero(weights)[0][-1])


def verify(target, ids, starts, uniforms, temps, draft=None, draft_temps=None):
    """(accepted, next_ids, chances) of the sequences; chances of rows of no sequence are NaN."""
    n, vocab = target.shape
    draft_temps = temps if draft_temps is None else draft_temps
    accepted, next_ids, chances = [], [], np.full(n, np.nan)
    for s in range(len(starts) - 1):
        a, b = int(starts[s]), int(starts[s + 1])
        if not 0 <= a < b <= n:
            accepted.append(0)
            next_ids.append(-1)
            continue
        chances[a] = 1.0
        stop = None
        for t in range(a + 1, b):
            x = int(ids[t])
            p = distribution(target[t - 1], temps[s])
            q = None if draft is None else distribution(draft[t], draft_temps[s])
            chance, yes = 0.0, False
            if p is not None and (draft is None or q is not None):
                inside = 0 <= x < vocab
                px = p[x] if inside else 0.0
                qx = 1.0 if draft is None else q[x] if inside else 0.0
                chance = min(1.0, px / max(qx, 1e-300)) if px > 0 else 0.0
                yes = np.float64(uniforms[t]) * qx < px
            chances[t] = chance
            if not yes and stop is None:
                stop = t
        some = stop is not None
        stop = b if stop is None else stop
        accepted.append(stop - 1 - a)
        p = distribution(target[stop - 1], temps[s])
        q = None
        if some:
            x = int(ids[stop])
            q = np.zeros(vocab) if draft is None else distribution(draft[stop], draft_temps[s])
            if draft is None and 0 <= x < vocab:
                q[x] = 1.0
        if p is None or (some and q is None):
            next_ids.append(-1)
            continue
        r = np.maximum(p - q, 0.0) if some else p
        next_ids.append(draw(r if r.sum() > 0 else p, uniforms[a]))
    return np.array(accepted), np.array(next_ids), chances
