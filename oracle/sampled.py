"""Oracle of the sampled verification of drafted tokens -- TEST INFRASTRUCTURE ONLY.

The definition in float64, one request at a time: softmax with the suppressed
ids left out, acceptance while ``u q(x) < p(x)``, next token by inverse
cumulative sum of ``max(p - q, 0)`` (or of ``p``) in id order.  The greedy tail
it generalises is ``dflash_mlx/engine/spec_epoch.py:2067-2072,2129``.
"""

from __future__ import annotations

import numpy as np


def distribution(row, z, suppressed=None):
    """Softmax of one row at temperature z; zeros where nothing can be drawn."""
    x = np.array(row, np.float64, copy=True)
    if suppressed is not None:
        x[np.asarray(suppressed, bool)] = -np.inf
    x[np.isnan(x)] = -np.inf
    m = x.max()
    if m == -np.inf:
        return np.zeros_like(x)
    if not z > 0:
        return (np.arange(x.size) == int(x.argmax())).astype(np.float64)
    if m == np.inf:
        w = (x == np.inf).astype(np.float64)
    else:
        w = np.exp((x - m) / np.float64(z))
    return w / w.sum()


def pick(w, u):
    """First id whose cumulative weight exceeds ``u`` of the total; -1 for none."""
    c = np.cumsum(w)
    if not c[-1] > 0:
        return -1
    over = np.nonzero(c > max(float(u), 0.0) * c[-1])[0]
    return int(over[0]) if over.size else int(np.nonzero(w > 0)[0][-1])


def verify_accept_sampled(logits, ids, accept_u, sample_u, draft=None, temperature=None, lens=None,
                          suppressed=None):
    """(accepted [B], token [B], draft_prob float64 [B, T-1])."""
    b, t, v = logits.shape
    acc, tok, prob = [], [], np.zeros((b, t - 1))
    for i in range(b):
        z = temperature[i]
        n = t - 1 if lens is None else int(lens[i])
        p = [distribution(logits[i, r], z, suppressed) for r in range(n + 1)]
        q = []
        for r in range(n):
            x = int(ids[i, r + 1])
            if draft is None or not z > 0:
                q.append((np.arange(v) == x).astype(np.float64))
            else:
                q.append(distribution(draft[i, r], z))
            prob[i, r] = p[r][x] if 0 <= x < v else 0.0
        a = 0
        while a < n:
            x = int(ids[i, a + 1])
            qx = q[a][x] if 0 <= x < v else 0.0
            if not float(accept_u[i, a]) * qx < prob[i, a]:
                break
            a += 1
        w = p[a]
        if a < n:
            left = np.maximum(p[a] - q[a], 0.0)
            w = left if left.sum() > 0 else p[a]
        acc.append(a)
        tok.append(pick(w, sample_u[i]))
    return np.array(acc, np.int32), np.array(tok, np.int32), prob
