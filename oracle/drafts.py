"""leafq_verify_drafts (include/leafq.h) from its definition in 64-bit floats: what
the GPU tests compare with."""
from __future__ import annotations

import numpy as np


def target(logits, temperature):
    """The distribution of one row, or None where it has none."""
    x = np.asarray(logits, dtype=np.float64).copy()
    x[np.isnan(x)] = -np.inf
    top = x.max()
    if top == -np.inf:
        return None
    if not temperature > 0:
        p = np.zeros_like(x)
        p[int(np.argmax(x == top))] = 1.0
        return p
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == top, 1.0, np.where(x == -np.inf, 0.0, np.exp((x - top) / float(temperature))))
    return w / w.sum()


def verify(logits, ids, parents, accept, sample, temperature, draft_probs=None):
    """Of one request: (path, tokens, margins), the margins being how far the nearest
    comparison of a child (relative to its sides) and of the draw (of the whole
    sum) were from turning out the other way."""
    n = len(ids)
    path, tokens, child, draw = [], [], np.inf, np.inf
    u = 0
    while n:
        path.append(u)
        own = target(logits[u], temperature)
        if own is None:
            tokens.append(-1)
            break
        greedy = not temperature > 0
        p, found = own, -1
        for c in range(u + 1, n):
            x = int(ids[c])
            if int(parents[c]) != u or not 0 <= x < len(own):
                continue
            if greedy:
                if own[x] == 1.0:
                    found = c
                    break
                continue
            if draft_probs is None:
                q = np.zeros_like(own)
                q[x] = 1.0
            else:
                q = np.asarray(draft_probs[u], dtype=np.float64)
                q = np.where(q > 0, q, 0.0)
            a, b = float(accept[c]) * q[x], p[x]
            child = min(child, abs(a - b) / max(a, b)) if max(a, b) > 0 else child
            if a < b:
                found = c
                break
            left = np.maximum(p - q, 0.0)
            p = left / left.sum() if left.sum() > 0 else own
        if found >= 0:
            tokens.append(int(ids[found]))
            u = found
            continue
        upto = np.cumsum(p)
        goal = min(max(float(sample), 0.0), 1 - 2.0 ** -24) * upto[-1]
        if not greedy:
            draw = np.abs(upto - goal).min() / upto[-1]
        drawn = int(np.searchsorted(upto, goal, side="right"))
        tokens.append(min(drawn, int(np.flatnonzero(p > 0)[-1])))
        break
    return path, tokens, (child, draw)
