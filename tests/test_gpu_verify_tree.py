"""Accept/resample over trees (``plh_verify_tree``) against the oracle, and rounds
of a small model that run the operators together (needs an MI355X).

Both sides work in float64 from the same values, in other orders of summation:
tokens and paths must be equal unless a uniform lies within 1e-12 of a border, the
bar of the chain's tests (none has)."""

from __future__ import annotations

import numpy as np
import pytest

import oracle
from oracle import tree as O
from pagellm_amd.cache import PagedCache, Rotary
from pagellm_amd.params import SamplingParams, make_rng
from pagellm_amd.speculative import verify_batch
from pagellm_amd.tree import DraftTree, TreeDecoder, tree_attention, verify_tree, verify_tree_step

pytestmark = pytest.mark.gpu


def _case(seed, counts, V, width, dtype, replacement, sharp=3.0, near=0.5):
    """Trees with children drawn from the draft's distributions."""
    g = np.random.default_rng(seed)
    N = sum(counts)
    z = sharp * g.standard_normal((N, V))
    soft = lambda x: np.exp(x - x.max(1, keepdims=True)) / np.exp(x - x.max(1, keepdims=True)).sum(1, keepdims=True)  # noqa: E731
    p, q = soft(z).astype(dtype), soft((1 - near) * z + near * sharp * g.standard_normal((N, V))).astype(dtype)
    tokens, parents, off = np.zeros(N, int), np.zeros(N, int), np.cumsum([0] + counts)
    for b, n in enumerate(counts):
        s = off[b]
        par = [-1] + [int(g.integers(max(0, (i - 1) // width - 1), (i - 1) // width + 1)) for i in range(1, n)]
        parents[s:s + n] = par
        for node in range(n):
            kids = [i for i in range(n) if par[i] == node]
            w = q[s + node].astype(np.float64)
            m = min(len(kids), int((w > 0).sum())) if not replacement else len(kids)
            draw = g.choice(V, m, replace=replacement, p=w / w.sum())
            for i, x in zip(kids, draw):
                tokens[s + i] = x
    return p, q, tokens, parents, off, g.random((len(counts), max(counts)))


def _check(res, p, q, tokens, parents, off, u, replacement):
    near = 0
    for b in range(len(off) - 1):
        s, e = off[b], off[b + 1]
        toks, path, used, gap = O.verify_tree(p[s:e], None if q is None else q[s:e], tokens[s:e], parents[s:e], u[b], replacement)
        n = len(path) - 1
        same = (list(res.tokens[b][: n + 1]) == toks and list(res.path[b][: n + 1]) == path and res.n_acc[b] == n
                and res.n_used[b] == used and np.all(res.tokens[b][n + 1:] == -1) and np.all(res.path[b][n + 1:] == -1))
        near += gap < 1e-6
        assert same or gap < 1e-12, (b, toks, path, used, gap, res.tokens[b], res.path[b], res.n_acc[b], res.n_used[b])
    return near


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("replacement", [False, True])
@pytest.mark.parametrize("V", [1, 2, 5, 65, 511, 512, 513, 4096, 32000, 50257])
def test_trees(V, replacement, dtype):
    counts = [1, 2, 3, 5, 8, 13, 21, 34, 64, 100, 7, 7] if V < 5000 else [1, 4, 9, 17, 30]
    total = 0
    for width, near in ((1, 0.5), (2, 0.5), (3, 0.9), (6, 1.0)):
        c = _case(V + width, counts, V, width, dtype, replacement, near=near)
        res = verify_tree(*c, replacement=replacement)
        total += _check(res, *c, replacement)
    print(f"[tree] V={V} {dtype} replacement={replacement}: {total} sequences within 1e-6 of a border", flush=True)


@pytest.mark.parametrize("V", [3, 65, 3333, 130000, 524288])
def test_drafts_without_distributions(V):
    """q None: drafts by rank of the target itself, and others."""
    counts = [1, 3, 9, 20]
    p, _, tokens, parents, off, u = _case(V, counts, V, 3, "float64", True)
    g = np.random.default_rng(V)
    for b in range(len(counts)):
        for i in range(off[b] + 1, off[b + 1]):
            row = off[b] + parents[i]
            tokens[i] = np.argsort(-p[row])[min(V - 1, int(g.integers(0, 3)))]
    res = verify_tree(p, None, tokens, parents, off, u)
    _check(res, p, None, tokens, parents, off, u, False)


def test_a_chain_is_the_batched_verify():
    g = np.random.default_rng(7)
    B, k, V = 40, 5, 1000
    p = g.dirichlet(np.full(V, 0.05), (B, k + 1))
    q = 0.6 * p[:, :k] + 0.4 * g.dirichlet(np.full(V, 0.05), (B, k))
    draft = np.array([[g.choice(V, p=q[b, i] / q[b, i].sum()) for i in range(k)] for b in range(B)])
    rngs = [np.random.default_rng(b) for b in range(B)]
    u = np.stack([np.random.default_rng(b).random(k + 1) for b in range(B)])
    toks, n = verify_batch(p, q, draft, rngs)
    qn = np.concatenate([q, np.zeros((B, 1, V))], 1).reshape(-1, V)
    res = verify_tree(p.reshape(-1, V), qn, np.concatenate([np.zeros((B, 1), int), draft], 1).reshape(-1),
                      np.tile(np.arange(-1, k), B), np.arange(0, B * (k + 1) + 1, k + 1), u)
    assert np.array_equal(res.tokens, toks) and np.array_equal(res.n_acc, n)
    for b in range(B):  # as many uniforms as the reference's loop draws
        h = np.random.default_rng(b)
        h.random(int(res.n_used[b]))
        assert h.random() == rngs[b].random()


def test_the_first_token_follows_the_target():
    """60 000 trees of one root and three siblings in one call: five standard
    deviations of a token's count."""
    g = np.random.default_rng(8)
    V, n = 6, 60000
    p, q = g.dirichlet(np.ones(V), 4), g.dirichlet(np.ones(V), 4)
    keys = np.log(q[0]) - np.log(-np.log(g.random((n, V))))
    kids = np.argsort(-keys, 1)[:, :3]
    tokens = np.concatenate([np.zeros((n, 1), int), kids], 1).reshape(-1)
    res = verify_tree(np.tile(p, (n, 1)), np.tile(q, (n, 1)), tokens, np.tile([-1, 0, 0, 0], n), np.arange(0, 4 * n + 1, 4),
                      g.random((n, 4)))
    count = np.bincount(res.tokens[:, 0], minlength=V)
    assert np.all(np.abs(count - n * p[0]) < 5 * np.sqrt(n * p[0] * (1 - p[0])))


def test_edges_of_the_rule():
    V = 600
    one = np.zeros(V)
    one[3] = 1.0
    flat = np.full(V, 1.0 / V)
    half = np.zeros(V)
    half[[3, 599]] = 0.5
    # the draft's token has no mass in the target: rejected, and drawn from what is left
    p, q = np.stack([half, flat, flat]), np.stack([flat, flat, flat])
    res = verify_tree(p, q, [0, 7, 8], [-1, 0, 0], [0, 3], [[0.0, 0.0, 0.7]])
    assert res.n_acc[0] == 0 and res.tokens[0, 0] == 599 and res.n_used[0] == 3
    # the draft's distribution is the target's: every first child is accepted
    res = verify_tree(np.stack([flat] * 4), np.stack([flat] * 4), [0, 5, 6, 7], [-1, 0, 1, 2], [0, 4], [[0.999999] * 4])
    assert res.n_acc[0] == 3 and res.path[0].tolist() == [0, 1, 2, 3]
    # a uniform of 1 rejects it, nothing is left, and the target itself is drawn from
    res = verify_tree(np.stack([half] * 3), np.stack([half] * 3), [0, 3, 599], [-1, 0, 0], [0, 3], [[1.0, 0.2, 0.6]])
    assert res.n_acc[0] == 0 and res.tokens[0, 0] == 3 and res.n_used[0] == 2
    # the same token twice among siblings is not accepted on what is no longer there
    res = verify_tree(np.stack([one, flat, flat]), np.stack([flat] * 3), [0, 9, 9], [-1, 0, 0], [0, 3], [[0.5, 0.0, 0.0]])
    assert res.n_acc[0] == 0 and res.tokens[0, 0] == 3
    # no mass at all: the last id
    res = verify_tree(np.zeros((1, V)), np.zeros((1, V)), [0], [-1], [0, 1], [[0.5]])
    assert res.tokens[0, 0] == V - 1


def test_device_calls_with_broken_sequences():
    """Tokens and offsets that no host check has seen: -1, and the others as ever."""
    import torch

    p, q, tokens, parents, off, u = _case(3, [6, 6, 6, 6], 700, 2, "float64", False)
    up = lambda x, t: torch.from_numpy(np.ascontiguousarray(x)).to("cuda", t)  # noqa: E731
    i32 = torch.int32

    def go(tokens, parents, off, q=q):
        return [x.cpu().numpy() for x in verify_tree(up(p, torch.float64), up(q, torch.float64), up(tokens, i32), up(parents, i32),
                                                     up(off, i32), up(u, torch.float64), max_nodes=6)]
    good = go(tokens, parents, off)
    for x in (-1, 700, 2**31 - 1):
        t = tokens.copy()
        t[7:12] = x
        got = go(t, parents, off)
        assert got[2][1] == -1 and got[3][1] == 0 and np.all(got[0][1] == -1) and np.all(got[1][1] == -1)
        for b in (0, 2, 3):
            assert all(np.array_equal(a[b], w[b]) for a, w in zip(got, good))
    for bad in ([0, 6, 6, 18, 24], [0, 6, 12, 25, 24], [0, 6, -5, 18, 24], [0, 6, 13, 18, 24]):
        got = go(tokens, parents, np.array(bad))
        assert got[2][1] == -1 or got[2][2] == -1
        assert all(np.array_equal(a[0], w[0]) for a, w in zip(got, good))
    par = parents.copy()
    par[6:12] = [-1, 5, 9, -7, 4, 100]  # never tested
    assert go(tokens, par, off)[2][1] == 0


def test_strides_streams_and_graphs():
    import torch

    p, q, tokens, parents, off, u = _case(4, [9, 20, 3], 5000, 3, "float32", False)
    up = lambda x, t: torch.from_numpy(np.ascontiguousarray(x)).to("cuda", t)  # noqa: E731
    wide = torch.full((32, 10007), 9.0, device="cuda")
    P, Q = wide[:, 1:5001], wide[:, 5003:10003]
    P.copy_(up(p, torch.float32))
    Q.copy_(up(q, torch.float32))
    args = [P, Q, up(tokens, torch.int32), up(parents, torch.int64), up(off, torch.int64), up(u, torch.float64)]
    want = verify_tree(*args, max_nodes=20)
    _check(type(want)(*(x.cpu().numpy() for x in want)), p, q, tokens, parents, off, u, False)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = verify_tree(*args, max_nodes=20)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = verify_tree(*args, max_nodes=20)
    for i in range(4):
        args[5].copy_(torch.rand(3, 20, dtype=torch.float64, device="cuda"))
        graph.replay()
        want = verify_tree(*args, max_nodes=20)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    with pytest.raises(NotImplementedError):
        verify_tree(P, Q, *args[2:5], torch.zeros((3, 257), dtype=torch.float64, device="cuda"), max_nodes=257)
    with pytest.raises(NotImplementedError):
        big = torch.zeros((1, 524289), device="cuda")
        verify_tree(big, None, [0], [-1], [0, 1], torch.zeros((1, 1), dtype=torch.float64, device="cuda"), max_nodes=1)


@pytest.mark.parametrize("dtype", ["float32", "float64"])
@pytest.mark.parametrize("V", [8193, 20000, 70001])
def test_results_do_not_depend_on_waits(V, dtype):
    """With no look for another workgroup's sums every workgroup computes all of
    them itself: the same bits; many sequences, so that some start late."""
    import torch

    from pagellm_amd import _native

    ctx = _native.Context()
    for replacement, with_q in ((False, True), (True, True), (False, False)):
        p, q, tokens, parents, off, u = _case(V, [40, 1, 7, 2] * 3, V, 4, dtype, replacement, near=1.0)
        many = lambda x: np.concatenate([x] * 8)  # noqa: E731
        n = off[-1]
        args = [many(p), many(q) if with_q else None, many(tokens), many(parents),
                np.concatenate([[0]] + [off[1:] + n * i for i in range(8)]), np.random.default_rng(1).random((96, 40))]
        up = lambda x, t: None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to("cuda", t)  # noqa: E731
        dt = getattr(torch, dtype)
        args = [up(x, t) for x, t in zip(args, (dt, dt, torch.int32, torch.int32, torch.int32, torch.float64))]
        want = verify_tree(*args, max_nodes=40, replacement=replacement, ctx=ctx)
        for looks in (0, 1, 64):
            ctx._check(ctx.lib.plh_set_option(ctx.handle, _native.PLH_OPT_TREE_LOOKS, looks))
            got = verify_tree(*args, max_nodes=40, replacement=replacement, ctx=ctx)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (looks, replacement, with_q)
    with pytest.raises(ValueError):
        ctx._check(ctx.lib.plh_set_option(ctx.handle, _native.PLH_OPT_TREE_LOOKS, -1))


def test_more_rejections_than_shared_sums():
    """A root with 60 children that are all rejected: passes past the shared ones."""
    V = 9000
    g = np.random.default_rng(2)
    q = g.dirichlet(np.ones(V), 61)
    p = np.zeros((61, V))
    p[:, 8500:] = 1 / 500
    kids = g.permutation(8000)[:60]
    u = g.random((1, 61))
    args = [p, q, np.concatenate([[0], kids]), np.array([-1] + [0] * 60), np.array([0, 61]), u]
    res = verify_tree(*args)
    _check(res, *args, False)
    assert res.n_used[0] == 61 and res.n_acc[0] == 0 and res.tokens[0, 0] >= 8500


@pytest.mark.parametrize("on_gpu", [False, True])
def test_a_round_from_logits_and_generators(on_gpu):
    """verify_tree_step against the oracle's probs and rule, Generators left where a
    loop of single draws leaves them."""
    import torch

    g = np.random.default_rng(9)
    V = 400
    trees = [DraftTree([1]), DraftTree([2, 3, 4, 5], [-1, 0, 0, 1]), DraftTree([7, 8, 9, 10, 11, 12], [-1, 0, 0, 2, 2, 4])]
    params = [SamplingParams(temperature=0.0), SamplingParams(temperature=0.8, top_k=30, repetition_penalty=1.3),
              SamplingParams(temperature=1.0, top_p=0.9)]
    ctx = [[5, 1], [9, 9, 30, 2], [7]]
    N = sum(map(len, trees))
    logits = (2 * g.standard_normal((N, V))).astype(np.float32)
    for t, s in zip(trees, (0, 1, 5)):
        for i in range(1, len(t)):
            logits[s + t.parents[i], t.tokens[i]] += 5.0
    q = g.dirichlet(np.full(V, 0.3), N)
    for rows in (None, q):
        rngs, mine = ([make_rng(s, 0) for s in (1, 2, 3)] for _ in range(2))
        x = torch.from_numpy(logits).cuda() if on_gpu else logits
        qq = torch.from_numpy(rows).cuda() if on_gpu and rows is not None else rows
        res = verify_tree_step(x, qq, trees, params, rngs, ctx)
        s = 0
        for b, t in enumerate(trees):
            p = np.stack([oracle.probs(logits[s + i], params[b], ctx[b] + t.path_to(i)) for i in range(len(t))])
            u = mine[b].bit_generator.state
            toks, path, used, gap = O.verify_tree(p, None if rows is None else rows[s:s + len(t)], t.tokens, t.parents,
                                                  mine[b].random(len(t)))
            mine[b].bit_generator.state = u
            mine[b].random(used)
            assert (res.emitted[b] == toks and res.n_acc[b] == len(path) - 1) or gap < 1e-12
            assert rngs[b].random() == mine[b].random()
            s += len(t)


class Model:
    """A small decoder of random weights with rotary positions and grouped heads,
    in float32 on the GPU; its attention is a step's."""

    def __init__(self, V=97, layers=2, heads=4, kv_heads=2, dim=32, seed=0):
        import torch

        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        D = heads * dim
        rnd = lambda *s: torch.randn(s, generator=g, device="cuda") / s[0] ** 0.5  # noqa: E731
        self.V, self.heads, self.kv_heads, self.dim, self.layers = V, heads, kv_heads, dim, layers
        self.embed, self.head = rnd(V, D) * V ** 0.5, 6 * rnd(D, V)
        self.w = [(rnd(D, (heads + 2 * kv_heads) * dim), rnd(D, D), rnd(D, 2 * D), rnd(2 * D, D)) for _ in range(layers)]
        self.rot = Rotary(dim)

    @staticmethod
    def norm(x):
        return x * (x.square().mean(1, keepdim=True) + 1e-5).rsqrt()

    def forward(self, tokens, attend):
        h = self.embed[tokens.long()]
        N, d = h.shape[0], self.dim
        for layer, (qkv, o, up, down) in enumerate(self.w):
            x = self.norm(h) @ qkv
            q, k, v = (t.view(N, -1, d) for t in x.split([self.heads * d, self.kv_heads * d, self.kv_heads * d], 1))
            h = h + attend(layer, q, k, v).reshape(N, -1) @ o
            h = h + (self.norm(h) @ up).relu() @ down
        return self.norm(h) @ self.head

    def step(self, s):
        return self.forward(s.tokens, lambda layer, q, k, v: s.attend(layer, q, k, v, self.rot))

    def alone(self, tokens):
        """Logits of one sequence's last token, attention in float64, nothing cached."""
        import torch

        n = len(tokens)

        def attend(layer, q, k, v):
            x = [a.double().cpu().numpy() for a in (q, k, v)]
            f = self.rot.inv_freq.cpu().numpy()
            x[0], x[1] = (O.rotate(a, np.arange(n), f) for a in x[:2])
            out = np.stack([O.attend_sequence(x[0][:, h], x[1][:, h * self.kv_heads // self.heads],
                                              x[2][:, h * self.kv_heads // self.heads], np.tril(np.ones((n, n), bool)),
                                              self.dim ** -0.5)[0] for h in range(self.heads)], 1)
            return torch.from_numpy(out).to("cuda", torch.float32)

        return self.forward(torch.tensor(tokens, device="cuda"), attend)[-1].cpu().numpy()


def _draft(g, model, context, n):
    """A tree of guesses: the model's own best tokens for the root, then random ones."""
    best = np.argsort(-model.alone(context))[:2]
    tokens, parents = [context[-1]], [-1]
    for i in range(1, n):
        parents.append(int(g.integers(0, i)))
        tokens.append(int(best[i % 2]) if parents[-1] == 0 else int(g.integers(0, model.V)))
        if parents[-1] > 0 and g.random() < 0.6:
            up, way = i, []
            node = parents[-1]
            while node > 0:
                way.append(tokens[node])
                node = parents[node]
            tokens[-1] = int(np.argmax(model.alone(context + way[::-1])))
    return DraftTree(tokens, parents)


def test_greedy_rounds_give_what_single_steps_give():
    """Prefill, rounds with trees, a fork, removals: greedy tokens are those of the
    model run from scratch, one token at a time."""
    model = Model()
    cache = PagedCache(model.layers, 64, 16, model.kv_heads, model.dim, "float32")
    dec = TreeDecoder(cache, model.step)
    g = np.random.default_rng(1)
    prompts = {"a": [5], "b": [int(t) for t in g.integers(0, 97, 21)], "c": [int(t) for t in g.integers(0, 97, 33)]}
    dec.prefill(list(prompts), list(prompts.values()))
    ctx = {k: list(v) for k, v in prompts.items()}
    params = SamplingParams(temperature=0.0)
    accepted = 0
    for r in range(5):
        if r == 2:
            cache.fork("b", "d")
            ctx["d"] = list(ctx["b"])
        if r == 4:
            cache.remove("c")
            del ctx["c"]
        keys = list(ctx)
        trees = [_draft(g, model, ctx[k], int(g.integers(1, 12))) for k in keys]
        emitted, n_acc, _ = dec.round(keys, trees, params, [make_rng(0, i) for i in range(len(keys))], [ctx[k] for k in keys])
        for key, toks in zip(keys, emitted):
            for t in toks:
                x = model.alone(ctx[key])
                assert x[t] >= x.max() - 1e-3 * np.abs(x).max(), (key, r)  # the best, up to float32's order of sums
                ctx[key].append(t)
            assert cache.length(key) == len(ctx[key]) - 1
        accepted += int(n_acc.sum())
    assert accepted > 5
    with pytest.raises(ValueError):
        dec.prefill(["a"], [[1]])
    with pytest.raises(RuntimeError):
        dec.prefill(["x", "y"], [[1] * 5000, [1]])
    assert "x" not in cache and "y" not in cache
    for key in list(ctx):
        cache.remove(key)
    assert cache.free_pages == 64


def test_a_failed_prefill_leaves_no_sequence():
    cache = PagedCache(1, 4, 16, 1, 8, "float32")

    def forward(step):
        raise OverflowError("no logits")

    dec = TreeDecoder(cache, forward)
    cache.add("old")
    for keys, prompts, error in [(["a", "b"], [[1, 2], [3]], OverflowError), (["a"], [range(100)], RuntimeError),
                                 (["a", "a"], [[1], [2]], ValueError), (["a", "old"], [[1], [2]], ValueError)]:
        with pytest.raises(error):
            dec.prefill(keys, prompts)
        assert len(cache) == 1 and cache.free_pages == 4


def test_sequences_have_generators_of_their_own():
    rng = make_rng(1, 0)
    trees = [DraftTree([1, 2]), DraftTree([3])]
    logits = np.random.default_rng(0).standard_normal((3, 8))
    with pytest.raises(ValueError):
        verify_tree_step(logits, None, trees, SamplingParams(), [rng, rng])


def test_sampled_rounds_run_with_penalties():
    model = Model(seed=3)
    cache = PagedCache(model.layers, 64, 16, model.kv_heads, model.dim, "float32")
    dec = TreeDecoder(cache, model.step)
    dec.prefill([0, 1], [[3, 4, 5], [6]])
    ctx, g = [[3, 4, 5], [6]], np.random.default_rng(2)
    params = [SamplingParams(temperature=0.9, top_k=20, repetition_penalty=1.2), SamplingParams(temperature=1.0, top_p=0.95)]
    rngs, mine = ([make_rng(s, 0) for s in (1, 2)] for _ in range(2))
    for _ in range(4):
        trees = [_draft(g, model, c, 8) for c in ctx]
        p = [np.stack([oracle.probs(model.alone(c + t.path_to(i)), prm, c + t.path_to(i)) for i in range(len(t))])
             for c, t, prm in zip(ctx, trees, params)]
        emitted, n_acc, _ = dec.round([0, 1], trees, params, rngs, ctx)
        for b, t in enumerate(trees):
            state = mine[b].bit_generator.state
            toks, path, used, gap = O.verify_tree(p[b], None, t.tokens, t.parents, mine[b].random(len(t)))
            mine[b].bit_generator.state = state
            mine[b].random(used)
            # the model's float32 sums run in other orders here and there
            assert emitted[b] == toks or gap < 1e-3
            if emitted[b] != toks:
                return
            ctx[b] += toks


def test_two_graphs_at_once():
    """Captured calls with workspaces of their own, replayed on two streams together."""
    import torch

    def verdicts(seed):
        p, q, tokens, parents, off, u = (torch.from_numpy(np.ascontiguousarray(x)).cuda()
                                         for x in _case(seed, [9, 16, 3], 20_000, 3, "float64", False))
        return lambda: verify_tree(p, q, tokens, parents, off, u, max_nodes=16)

    def outputs(seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        k, v = (torch.randn(300, 2, 16, 128, generator=g, device="cuda").half() for _ in range(2))
        x = torch.randn(50, 8, 128, generator=g, device="cuda").half()
        table = torch.arange(300, dtype=torch.int32, device="cuda").view(2, 150)
        lens, off = (torch.tensor(n, dtype=torch.int32, device="cuda") for n in ([2000 + seed, 40], [0, 20, 50]))
        return lambda: (tree_attention(x, k, v, table, lens, off, max_nodes=30, max_len=2100),)

    for make in (verdicts, outputs):
        calls = [make(1), make(2)]
        want = [[x.clone() for x in call()] for call in calls]
        torch.cuda.synchronize()
        streams, graphs, got = [torch.cuda.Stream() for _ in calls], [], []
        for call, s in zip(calls, streams):
            graphs.append(torch.cuda.CUDAGraph())
            with torch.cuda.graph(graphs[-1], stream=s):
                got.append(call())
        for _ in range(5):
            for graph, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    graph.replay()
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert all(torch.equal(x, y) for x, y in zip(a, b))
                for x in a:
                    x.fill_(3)
            for call, b in zip(calls, want):  # eager calls in between
                assert all(torch.equal(x, y) for x, y in zip(call(), b))
            torch.cuda.synchronize()
