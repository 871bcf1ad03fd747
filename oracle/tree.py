"""CPU oracle for speculation with trees over a paged cache: test infrastructure only.

Plain float64 numpy, one sequence (and head) at a time.  The accept/resample rule
is ``src/pagellm/engine/speculative.py:38-60`` applied to a node's children in
turn; the reference drafts chains.
"""

from __future__ import annotations

import numpy as np


def verify_tree(p, q, tokens, parents, uniforms, replacement=False):
    """One sequence's tree: p, q [T, V] (q None: drafts that are their draft's only
    choice).  Returns (emitted tokens, path from 0 on, uniforms used, gap): gap is
    the smallest distance of a uniform to a border of its test or draw."""
    p = np.asarray(p, dtype=np.float64)
    T, V = p.shape
    cur, t, path, toks, gap = 0, 0, [0], [], np.inf
    r, s, tested = p[0], None if q is None else np.asarray(q[0], dtype=np.float64), False
    with np.errstate(divide="ignore", invalid="ignore"):
        for i in range(1, T):
            if parents[i] != cur:
                continue
            x = int(tokens[i])
            sx = 1.0 if q is None else s[x]
            thr = r[x] / sx if r[x] > 0 or not tested else np.float64(0.0)
            thr = min(1.0, thr) if not np.isnan(thr) else 1.0
            u = float(uniforms[t])
            t += 1
            gap = min(gap, abs(u - thr))
            if u < thr:
                cur, tested = i, False
                path.append(i)
                toks.append(x)
                r, s = p[i], None if q is None else np.asarray(q[i], dtype=np.float64)
                continue
            tested = True
            if q is None:
                left = r.copy()
                left[x] = max(r[x] - 1.0, 0.0)
            else:
                left = np.maximum(r - s, 0.0)
            if left.sum() <= 0:
                r = p[cur]
                break
            r = left / left.sum()
            if q is not None and not replacement:
                s = s.copy()
                s[x] = 0.0
                s = s / s.sum()
    c = np.cumsum(r)
    u = float(uniforms[t])
    toks.append(int(min(np.searchsorted(c, u * c[-1], side="right"), V - 1)))
    return toks, path, t + 1, min(gap, float(np.min(np.abs(c / c[-1] - u))))


def rotate(x, positions, inv_freq, interleaved=False, factor=1.0):
    """x [N, heads, D] with its pairs turned, in float64."""
    y = np.array(x, dtype=np.float64)
    R = len(inv_freq)
    a = np.asarray(positions, dtype=np.float64)[:, None] * np.asarray(inv_freq, dtype=np.float64)
    c, s = factor * np.cos(a)[:, None], factor * np.sin(a)[:, None]
    first, second = (slice(0, 2 * R, 2), slice(1, 2 * R, 2)) if interleaved else (slice(0, R), slice(R, 2 * R))
    u, v = y[..., first].copy(), y[..., second].copy()
    y[..., first], y[..., second] = u * c - v * s, v * c + u * s
    return y


def attend_sequence(q, k, v, sees, scale):
    """One sequence and head: q [T, D], k, v [L, D], sees bool [T, L].  Returns
    (out [T, D], lse [T], spread [T, D], top [T]): spread is sum w |v| / sum w, and
    top the largest scale * sum |q| |k| that a row sees, for error bounds."""
    q, k, v = (np.asarray(x, dtype=np.float64) for x in (q, k, v))
    T, D = q.shape
    out, lse = np.zeros((T, D)), np.full(T, -np.inf)
    spread, top = np.zeros((T, D)), np.zeros(T)
    with np.errstate(invalid="ignore", over="ignore"):
        for i in range(T):
            at = np.flatnonzero(sees[i])
            if not at.size:
                continue
            x = scale * (k[at] @ q[i])
            m = x.max()
            w = np.exp(x - m)
            out[i] = (w[:, None] * v[at]).sum(0) / w.sum()
            spread[i] = (w[:, None] * np.abs(v[at])).sum(0) / w.sum()
            lse[i] = m + np.log(w.sum())
            # a score of -inf is a weight of exactly 0 however it is computed: no error
            top[i] = (scale * (np.abs(k[at]) @ np.abs(q[i])))[x > -np.inf].max(initial=0.0)
    return out, lse, spread, top


def sees_of(length: int, nodes: int, visible=None) -> np.ndarray:
    """bool [nodes, length + nodes]: which keys each node sees (visible: words of
    bits, or None for a chain)."""
    s = np.ones((nodes, length + nodes), dtype=bool)
    for i in range(nodes):
        if visible is None:
            s[i, length:] = np.arange(nodes) <= i
        else:
            s[i, length:] = [(int(visible[i]) >> j) & 1 == 1 for j in range(nodes)]
    return s
