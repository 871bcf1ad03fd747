"""CPU oracle for products with e4m3 weights: test infrastructure only.

e4m3 here is OCP's: 4 exponent bits, 3 of mantissa, no infinities, largest
value 448, steps of 2^-9 below 2^-6.  float64 numpy; pinned by
``tests/test_oracle_logits.py`` against the table of all 256 codes.
"""

from __future__ import annotations

import numpy as np

BLOCK = 128


def decode(codes) -> np.ndarray:
    """float64 values of e4m3 codes (uint8)."""
    c = np.asarray(codes, dtype=np.uint8).astype(np.int64)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c & 128, -v, v)


def round_e4m3(x) -> np.ndarray:
    """The e4m3 value nearest to each x (|x| <= 448 or NaN), ties to even."""
    x = np.asarray(x, dtype=np.float64)
    _, e = np.frexp(np.abs(np.where(np.isnan(x), 0.0, x)))
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.round(x / step) * step


def block_scale(amax) -> np.ndarray:
    """The smallest power of two s >= 2^-126 with amax <= 448 s."""
    amax = np.asarray(amax, dtype=np.float64)
    m, e = np.frexp(amax)  # amax = m 2^e, 448 = 0.875 * 2^9
    e = np.where(amax > 0, np.where(m > 0.875, e - 8, e - 9), -126)
    return np.ldexp(1.0, np.maximum(e, -126))


def round_rows(y) -> np.ndarray:
    """Rows [N, D] (float32 values) rounded in blocks of 128 of a row: the values
    their codes and scales stand for.  A row with NaN or infinity becomes NaN."""
    y = np.asarray(y, dtype=np.float64)
    out = np.empty_like(y)
    bad = ~np.isfinite(y).all(axis=1)
    for k in range(0, y.shape[1], BLOCK):
        b = np.where(np.isfinite(y[:, k:k + BLOCK]), y[:, k:k + BLOCK], 0.0)
        s = block_scale(np.abs(b).max(axis=1, keepdims=True))
        out[:, k:k + BLOCK] = round_e4m3(b / s) * s
    out[bad] = np.nan
    return out


def round_matrix(w) -> np.ndarray:
    """A matrix [V, D] rounded in blocks of 128 x 128; NaN and infinities become NaN."""
    w = np.asarray(w, dtype=np.float64)
    out = np.empty_like(w)
    for v in range(0, w.shape[0], BLOCK):
        for k in range(0, w.shape[1], BLOCK):
            b = w[v:v + BLOCK, k:k + BLOCK]
            s = block_scale(np.max(np.abs(b), initial=0.0, where=np.isfinite(b)))
            out[v:v + BLOCK, k:k + BLOCK] = np.where(np.isfinite(b), round_e4m3(np.where(np.isfinite(b), b, 0) / s) * s,
                                                     np.nan)
    return out


def norm_rows(x, norm, eps: float) -> np.ndarray:
    """rms_norm in float64, rounded once to float32 (as float64 values)."""
    x = np.asarray(x, dtype=np.float64)
    r = 1.0 / np.sqrt((x * x).mean(axis=1, keepdims=True) + eps)
    return (x * r * np.asarray(norm, dtype=np.float64)).astype(np.float32).astype(np.float64)


def linear(x, w, norm=None, eps: float = 1e-5):
    """(out, bound): the product of the rounded rows with the matrix w [V, D] (the
    values its codes stand for), and sum |a| |w|, in float64."""
    y = np.asarray(x, dtype=np.float64) if norm is None else norm_rows(x, norm, eps)
    a = round_rows(y)
    w = np.asarray(w, dtype=np.float64)
    return a @ w.T, np.abs(a) @ np.abs(w).T
