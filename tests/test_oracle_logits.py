"""Pins the oracles of logits processing, log probabilities and e4m3 products
(``oracle/logits.py``, ``oracle/fp8.py``) on the CPU, against loops over single
tokens, math.fsum and the table of all e4m3 codes."""

from __future__ import annotations

import math

import numpy as np
import pytest

from oracle import fp8, logits


@pytest.mark.parametrize("seed", range(4))
def test_process_row_against_a_loop(seed):
    g = np.random.default_rng(seed)
    V = 70
    x = g.normal(0, 3, V)
    hist = g.integers(-3, V + 3, 40)
    bias = [(int(t), float(v)) for t, v in zip(g.integers(0, V, 10), g.normal(0, 2, 10))]
    words = g.integers(0, 2**32, 3, dtype=np.uint64).astype(np.uint32)
    got = logits.process_row(x, history=hist, out_start=15, rep=1.3, freq=0.5, pres=0.25, bias=bias, mask=words)
    for t in range(V):
        v = x[t]
        for i, b in reversed(bias):
            if i == t:
                v += b
                break
        if t in hist:
            v = v / 1.3 if v > 0 else v * 1.3
        n = sum(int(i) == t for i in hist[15:])
        if n > 0:
            v -= 0.5 * n + 0.25
        if not (int(words[t // 32]) >> (t % 32)) & 1:
            v = -math.inf
        assert got[t] == pytest.approx(v, rel=1e-15) or got[t] == v
    assert np.array_equal(logits.process_row(x), x)


def test_order_and_logprobs():
    x = np.array([1.0, -np.inf, 3.0, 3.0, -0.0, 0.0, np.nan])
    assert list(logits.order(x)) == [6, 2, 3, 0, 4, 5, 1]
    assert np.isnan(logits.logprobs_row(x)).all()
    y = x[:6]
    p = [math.exp(v) for v in y]
    ref = [v - math.log(math.fsum(p)) for v in y]
    np.testing.assert_allclose(logits.logprobs_row(y), ref, rtol=1e-14)
    assert np.all(logits.logprobs_row(np.full(5, -np.inf)) == -np.inf)
    assert np.isnan(logits.logprobs_row(np.array([1.0, np.inf]))).all()


def test_e4m3_table_and_rounding():
    v = fp8.decode(np.arange(256))
    fin = np.sort(np.unique(v[np.isfinite(v)]))
    assert fin.size == 253 and fin[-1] == 448 and fin[0] == -448 and np.isnan(v[[127, 255]]).all()
    assert v[0x38] == 1.0 and v[1] == 2.0 ** -9 and v[8] == 2.0 ** -6
    g = np.random.default_rng(0)
    x = np.concatenate([fin, (fin[1:] + fin[:-1]) / 2, g.uniform(-448, 448, 2000), g.normal(0, 0.02, 2000)])
    got = fp8.round_e4m3(x)
    pos = {float(t): i for i, t in enumerate(v[:127])}  # a value's code: its last bit says even or odd
    for a, b in zip(x, got):
        d = np.abs(fin - a)
        near = fin[d == d.min()]
        assert b in near
        if near.size == 2:
            assert pos[abs(float(b))] % 2 == 0
    # a rounding is off by at most half a step
    assert np.all(np.abs(got - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10))


def test_block_scales():
    for a in (448.0, 448.0 * (1 + 2**-23), 1.0, 3e38, 1e-30, 2.0 ** -149, 0.0, 447.9, 225.0, 224.0):
        s = float(fp8.block_scale(a))
        assert math.frexp(s)[0] == 0.5 and a <= 448 * s
        assert s == 2.0 ** -126 or a > 448 * s / 2


def test_linear_against_fsum():
    g = np.random.default_rng(1)
    x, w, norm = g.normal(0, 1, (3, 200)), fp8.round_matrix(g.normal(0, 0.02, (5, 200))), 1 + 0.1 * g.normal(0, 1, 200)
    got, bound = fp8.linear(x, w, norm, 1e-5)
    for n in range(3):
        r = 1 / math.sqrt(math.fsum(v * v for v in x[n]) / 200 + 1e-5)
        y = np.array([float(np.float32(x[n, k] * r * norm[k])) for k in range(200)])
        a = fp8.round_rows(y[None])[0]
        for k in range(200):
            s = float(fp8.block_scale(np.abs(y[k // 128 * 128:k // 128 * 128 + 128]).max()))
            assert abs(a[k] - y[k]) <= max(2.0 ** -4 * abs(y[k]), s * 2.0 ** -10)
        for v in range(5):
            assert got[n, v] == pytest.approx(math.fsum(a * w[v]), rel=1e-12, abs=1e-15)
            assert bound[n, v] == pytest.approx(math.fsum(np.abs(a * w[v])), rel=1e-12)
