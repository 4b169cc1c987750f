"""Verification of drafted tokens, one sequence after the other in 64 bits (test infrastructure)."""

from __future__ import annotations

import numpy as np

NO_TOKEN = 0xFFFFFFFF


def weights(row, temperature):
    """Relative probabilities of a row of logits; all zero where nothing is above -inf."""
    x = np.asarray(row, np.float32).astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return np.zeros(len(x))
    if not temperature > 0:
        w = np.zeros(len(x))
        w[int(x.argmax())] = 1.0
        return w
    with np.errstate(all="ignore"):
        w = np.exp((x - top) / float(temperature))
    return np.where(x == top, 1.0, np.where(x > -np.inf, np.nan_to_num(w), 0.0))


def draw(w, v):
    """The first index whose cumulative weight exceeds v times the whole; the last with any weight
    where none does."""
    c = np.cumsum(w)
    hit = np.nonzero((c > float(v) * c[-1]) & (w > 0))[0]
    some = np.nonzero(w > 0)[0]
    return int(hit[0]) if len(hit) else int(some[-1]) if len(some) else NO_TOKEN


def verify(logits, row_off, drafts, u, v, draft_logits=None, temperature=None):
    """(accepted, next) of every sequence."""
    accepted, nxt, d = [], [], 0
    for s in range(len(row_off) - 1):
        t = 1.0 if temperature is None else temperature[s]
        rows = logits[row_off[s]:row_off[s + 1]]
        k, n, rest = len(rows) - 1, 0, None
        while n < k:
            x = int(drafts[d + n])
            wp = weights(rows[n], t)
            p = wp / wp.sum() if wp.any() else wp
            if draft_logits is None or not t > 0:
                q = np.zeros(len(p))
                if x < len(q):
                    q[x] = 1.0
            else:
                wq = weights(draft_logits[d + n], t)
                q = wq / wq.sum() if wq.any() else wq
            if x < len(p) and (p[x] > 0 if not t > 0 else float(u[d + n]) * q[x] < p[x]):
                n += 1
                continue
            rest = np.maximum(p - q, 0.0)
            if not t > 0 or not rest.any():
                rest = p
            break
        if rest is None:
            rest = weights(rows[k], t)
        accepted.append(n)
        nxt.append(draw(rest, v[s] if t > 0 else 0.0))
        d += k
    return np.array(accepted, np.uint32), np.array(nxt, np.uint32)
