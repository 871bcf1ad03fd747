"""CPU oracle for logits processing and log probabilities: test infrastructure only.

Plain float64 numpy, one row at a time.  The repetition rule is
``src/pagellm/engine/sampling.py:52-62``; the reference has no counterpart for
the rest, which is pinned by ``tests/test_oracle_logits.py`` against loops over
single tokens.
"""

from __future__ import annotations

import numpy as np


def process_row(x, *, history=(), out_start=0, rep=1.0, freq=0.0, pres=0.0, bias=(), mask=None) -> np.ndarray:
    """The processed row in float64.  ``bias`` is (id, value) pairs, of which the
    last of an id counts; ``mask`` the row's 32-bit words or None.  Ids outside
    the vocabulary count for no token."""
    y = np.asarray(x, dtype=np.float64).copy()
    V = y.size
    for t, v in dict((int(t), float(v)) for t, v in bias).items():
        if 0 <= t < V:
            y[t] += v
    hist = np.asarray(history, dtype=np.int64).reshape(-1)
    outputs = hist[out_start:]
    hist, outputs = hist[(hist >= 0) & (hist < V)], outputs[(outputs >= 0) & (outputs < V)]
    if rep != 1.0 or freq != 0.0 or pres != 0.0:
        seen = np.unique(hist)
        with np.errstate(invalid="ignore", over="ignore"):
            y[seen] = np.where(y[seen] > 0, y[seen] / rep, y[seen] * rep)
            ids, n = np.unique(outputs, return_counts=True)
            y[ids] -= freq * n + pres
    if mask is not None:
        y[~allowed(mask, V)] = -np.inf
    return y


def touched(V, *, history=(), bias=(), mask=None) -> np.ndarray:
    """bool [V]: the tokens that some rule may change."""
    t = np.zeros(V, dtype=bool)
    ids = np.concatenate([np.asarray(history, dtype=np.int64).reshape(-1),
                          np.asarray([i for i, _ in bias], dtype=np.int64)])
    t[ids[(ids >= 0) & (ids < V)]] = True
    return t | (~allowed(mask, V) if mask is not None else False)


def allowed(mask, V: int) -> np.ndarray:
    words = np.asarray(mask).astype(np.int64) & 0xFFFFFFFF
    t = np.arange(V)
    return (words[t // 32] >> (t % 32)) & 1 == 1


def order(x) -> np.ndarray:
    """Token ids by logit descending, NaN first, then by id ascending."""
    x = np.asarray(x, dtype=np.float64) + 0.0
    return np.lexsort((np.arange(x.size), -np.where(np.isnan(x), 0.0, x), ~np.isnan(x)))


def logprobs_row(x) -> np.ndarray:
    """x - logsumexp(x) in float64; a row of -inf only gives -inf, one that
    holds NaN or +inf only NaN."""
    x = np.asarray(x, dtype=np.float64)
    if np.all(x == -np.inf):
        return np.full(x.size, -np.inf)
    if np.any(np.isnan(x)) or np.any(x == np.inf):
        return np.full(x.size, np.nan)
    m = x.max()
    return (x - m) - np.log(np.exp(x - m).sum())


def logprobs_error(x) -> float:
    """Bound of the error of a float32 row's log probabilities beside their own
    rounding: each exponential of d = x - m is computed in float32 from the
    rounded d (2^-24 |d|), its rounded product with log2 e (another 2^-24 |d|,
    and log2 e's own 2^-25 |d|) and an exponential right to 2^-23; the sum of
    these relative errors weighted by the exponentials bounds the sum's."""
    x = np.asarray(x, dtype=np.float64)
    x = x[np.isfinite(x)]
    d = x - x.max()
    e = np.exp(d)
    return float(2.0 ** -23 * (1 + 1.25 * (e * np.abs(d)).sum() / e.sum())) + 1e-12
