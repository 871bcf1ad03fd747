"""The tree oracle: a chain is the reference's verify; siblings keep the target's
law; rotation and attention against loops over single values."""

from __future__ import annotations

import math

import numpy as np
import pytest

import oracle
from oracle import tree as O


def _dist(g, n, V):
    x = g.random((n, V)) ** 3
    return x / x.sum(1, keepdims=True)


@pytest.mark.parametrize("k", [0, 1, 3, 6])
def test_a_chain_is_verify(k):
    g = np.random.default_rng(k)
    for _ in range(300):
        p, q = _dist(g, k + 1, 9), _dist(g, k + 1, 9)
        draft = g.integers(0, 9, k)
        u = g.random(k + 1)
        want, n = oracle.verify(p, q, [int(t) for t in draft], oracle.ScriptedRNG(list(u)))
        toks, path, used, _ = O.verify_tree(p, q, [0, *draft], np.arange(-1, k), u)
        assert toks == want and len(path) == n + 1 and used == min(n + 1, k) + 1


@pytest.mark.parametrize("replacement", [False, True])
def test_siblings_keep_the_target_law(replacement):
    """The first emitted token follows p whatever the draft: 40 000 trials, five
    standard deviations of a token's count."""
    g = np.random.default_rng(5)
    V, w, n = 5, 3, 40000
    p, q = _dist(g, 1 + w, V), _dist(g, 1 + w, V)
    count = np.zeros(V)
    for _ in range(n):
        kids = g.choice(V, w, replace=replacement, p=q[0])
        toks, *_ = O.verify_tree(p, q, [0, *kids], [-1] + [0] * w, g.random(w + 1), replacement)
        count[toks[0]] += 1
    assert np.all(np.abs(count - n * p[0]) < 5 * np.sqrt(n * p[0] * (1 - p[0])))


def test_only_choices_keep_the_target_law():
    g = np.random.default_rng(6)
    p = _dist(g, 3, 6)
    count = np.zeros(6)
    for _ in range(20000):
        toks, *_ = O.verify_tree(p, None, [0, 4, 1], [-1, 0, 0], g.random(3))
        count[toks[0]] += 1
    assert np.all(np.abs(count - 20000 * p[0]) < 5 * np.sqrt(20000 * p[0] * (1 - p[0])))


def test_a_node_of_a_rejected_branch_is_passed_over():
    p = np.eye(4)[[2, 0, 1, 3]]
    q = np.full((4, 4), 0.25)
    toks, path, used, _ = O.verify_tree(p, q, [0, 1, 2, 0], [-1, 0, 0, 1], [0.5] * 4)
    assert toks == [2, 1] and path == [0, 2] and used == 3


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotate(interleaved):
    g = np.random.default_rng(1)
    x, f = g.standard_normal((3, 2, 8)), [1.0, 0.3, 0.01]
    y = O.rotate(x, [0, 7, 100], f, interleaved, 1.5)
    for n, pos in enumerate([0, 7, 100]):
        for h in range(2):
            assert np.array_equal(y[n, h, 6:], x[n, h, 6:])
            for i, w in enumerate(f):
                a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + 3)
                z = 1.5 * complex(x[n, h, a], x[n, h, b]) * complex(math.cos(pos * w), math.sin(pos * w))
                assert abs(complex(y[n, h, a], y[n, h, b]) - z) < 1e-13


def test_attention_by_loops():
    g = np.random.default_rng(2)
    q, k, v = g.standard_normal((3, 4)), g.standard_normal((6, 4)), g.standard_normal((6, 4))
    sees = O.sees_of(3, 3, [1, 3, 5])
    assert sees.tolist() == [[True] * 3 + r for r in ([True, False, False], [True, True, False], [True, False, True])]
    out, lse, _, _ = O.attend_sequence(q, k, v, sees, 0.5)
    for i in range(3):
        w = [math.exp(0.5 * sum(a * b for a, b in zip(q[i], k[j]))) if sees[i, j] else 0.0 for j in range(6)]
        assert abs(lse[i] - math.log(math.fsum(w))) < 1e-13
        for d in range(4):
            assert abs(out[i, d] - math.fsum(w[j] * v[j, d] for j in range(6)) / math.fsum(w)) < 1e-13
    out, lse, _, _ = O.attend_sequence(q[:1], k[:0], v[:0], np.zeros((1, 0), bool), 1.0)
    assert not out.any() and lse[0] == -np.inf
