"""Logits processing (``plh_process_logits``) and log probabilities
(``plh_logprobs``) against the float64 oracle (needs an MI355X).

Tolerances.  A processed float32 token is computed in float64 and rounded once:
half a step, 2^-24 of the value, and the float64 steps' 2^-53 of each magnitude
on the way; a float64 one has the latter only (at most five of them).  Tokens no
rule touches keep their bits.  Log probabilities: ``oracle.logits.logprobs_error``
and one rounding; ids, ranks and order are exact."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import logits as O
from pagellm_amd import _native
from pagellm_amd.logits import LogitRules, pack_mask, process_logits, token_logprobs
from pagellm_amd.params import SamplingParams

pytestmark = pytest.mark.gpu

DTYPES = [np.float32, np.float64]
# one token; around a mask word; a quad's tail; around a chunk of 8192; several chunks; odd and even
SIZES = [1, 2, 31, 32, 33, 65, 1000, 8191, 8192, 8193, 16387, 50257]


def _tol(ref, mag, dt):
    half = 2.0 ** -24 if dt == np.float32 else 0.0
    with np.errstate(invalid="ignore"):
        return np.abs(ref) * half + 5 * 2.0 ** -53 * mag + 2.0 ** -149


def _case(seed, B, V, dt):
    g = np.random.default_rng(seed)
    x = g.normal(0, 3, (B, V)).astype(dt)
    # (repetition, rules, history length, prompt length, mask) in turn, neutral ones among them
    kinds = [
        (1.0, LogitRules(), 30, 10, None),
        (1.3, LogitRules(0.5, 0.25), 200, 120, "half"),
        (0.8, LogitRules(), 50, 0, None),
        (1.0, LogitRules(0.0, -0.7, {int(t): float(v) for t, v in zip(g.integers(0, V, 9), g.normal(0, 2, 9))}), 40, 5,
         "few"),
        (1.1, LogitRules(-0.3, 0.0, {0: 1.0, V - 1: -np.inf}), 0, 0, "none"),
        (1.2, LogitRules(0.1, 0.1, {int(t): 0.5 for t in range(min(V, 500))}), 300, 300, "all"),
    ]
    rows = [kinds[b % len(kinds)] for b in range(B)]
    hist = [g.integers(0, V, k[2]) // (1 + b % 3) for b, k in enumerate(rows)]
    masks = []
    for k in rows:
        if k[4] is None:
            masks.append(None)
        else:
            share = {"half": 0.5, "few": 3 / V, "none": -1.0, "all": 2.0}[k[4]]
            masks.append(pack_mask(g.random(V) < share, V))
    return x, rows, hist, masks


def _expected(x, rows, hist, masks):
    ref, mag, touched = np.empty(x.shape), np.empty(x.shape), np.zeros(x.shape, dtype=bool)
    for b, (rep, rule, _, plen, _) in enumerate(rows):
        bias = list(rule.logit_bias.items())
        active = rep != 1.0 or rule.penalises
        ref[b] = O.process_row(x[b], history=hist[b], out_start=plen, rep=rep, freq=rule.frequency_penalty,
                               pres=rule.presence_penalty, bias=bias, mask=masks[b])
        touched[b] = O.touched(x.shape[1], history=hist[b] if active else (), bias=bias, mask=masks[b])
        most = max([abs(v) for _, v in bias if np.isfinite(v)], default=0.0)
        mag[b] = (np.abs(x[b]) + most) * max(rep, 1 / rep) + abs(rule.frequency_penalty) * len(hist[b]) + \
            abs(rule.presence_penalty)
    return ref, mag, touched


def _check(got, x, rows, hist, masks):
    ref, mag, touched = _expected(x, rows, hist, masks)
    assert got.shape == x.shape and got.dtype == x.dtype
    bits = np.uint32 if x.dtype == np.float32 else np.uint64
    assert np.array_equal(got.view(bits)[~touched], x.view(bits)[~touched])
    assert np.array_equal(np.isneginf(got), np.isneginf(ref))
    fin = np.isfinite(ref)
    err = np.abs(got[fin].astype(np.float64) - ref[fin])
    assert np.all(err <= _tol(ref, mag, x.dtype)[fin]), float(err.max())


def _run_numpy(x, rows, hist, masks):
    have = [b for b, m in enumerate(masks) if m is not None]
    words = np.stack([masks[b] for b in have]) if have else None
    at = [have.index(b) if b in have else None for b in range(len(rows))] if have else None
    return process_logits(x, [k[1] for k in rows], [SamplingParams(repetition_penalty=k[0]) for k in rows], hist,
                          prompt_lens=[k[3] for k in rows], masks=words, mask_rows=at)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V", SIZES)
def test_process_matches_oracle(V, dt):
    print(f"[process] V={V} {dt.__name__}", flush=True)
    x, rows, hist, masks = _case(V, 7, V, dt)
    _check(_run_numpy(x, rows, hist, masks), x, rows, hist, masks)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V,pad,shift", [(65, 3, 1), (8193, 5, 3), (50257, 0, 0), (16384, 4, 1)])
def test_process_torch_strides_in_place_and_not(V, pad, shift, dt):
    """Rows that start anywhere (element alignment only); nothing outside the
    rows is written; in place gives the same bits."""
    import torch

    print(f"[process] strides V={V} {dt.__name__}", flush=True)
    B = 6
    x, rows, hist, masks = _case(V + 1, B, V, dt)
    want = _run_numpy(x, rows, hist, masks)
    buf = torch.full((B + 1, V + pad + shift), 77.0, dtype=getattr(torch, dt.__name__), device="cuda")
    view = buf[:B, shift:shift + V]
    view.copy_(torch.from_numpy(x))
    words = torch.from_numpy(np.stack([m if m is not None else pack_mask(np.ones(V, bool), V) for m in masks]).view(np.int32))
    wide = torch.zeros((B, words.shape[1] + 2), dtype=torch.int32, device="cuda")
    wide[:, :words.shape[1]] = words.cuda()
    args = dict(rules=[k[1] for k in rows], params=[SamplingParams(repetition_penalty=k[0]) for k in rows],
                contexts=[h.tolist() for h in hist], prompt_lens=[k[3] for k in rows], masks=wide[:, :words.shape[1]])
    got = process_logits(view, **args)
    obuf = torch.full((B, V + 7), 5.0, dtype=buf.dtype, device="cuda")
    process_logits(view, out=obuf[:, 3:3 + V], **args)
    same = process_logits(view, out=view, **args)
    assert same is view
    for t in (got, obuf[:, 3:3 + V], view):
        assert np.array_equal(t.cpu().numpy(), want)
    assert bool((obuf[:, :3] == 5).all()) and bool((obuf[:, 3 + V:] == 5).all())
    assert bool((buf[B] == 77).all()) and bool((buf[:, :shift] == 77).all()) and bool((buf[:, shift + V:] == 77).all())


@pytest.mark.parametrize("dt", DTYPES)
def test_process_infinities_and_nan(dt):
    """Masked places hold -inf whatever stood there; elsewhere infinities and
    NaN follow the formula; a row may keep nothing."""
    V = 300
    x = np.random.default_rng(0).normal(0, 1, (4, V)).astype(dt)
    low = np.finfo(dt).min
    x[:, :8] = [np.nan, np.inf, -np.inf, low, np.nan, np.inf, -np.inf, low]
    allow = np.ones(V, dtype=bool)
    allow[:4] = False
    words = np.stack([pack_mask(allow, V), pack_mask([], V)])
    rule = LogitRules(0.5, 0.0, {5: -1.0, 6: 1.0})
    got = process_logits(x, rule, SamplingParams(repetition_penalty=1.5), [[1, 2, 5, 6, 7]] * 4, masks=words,
                         mask_rows=[0, 1, None, 0])
    assert np.all(np.isneginf(got[1]))
    for b in (0, 3):
        assert np.all(np.isneginf(got[b, :4])) and np.isnan(got[b, 4]) and got[b, 5] == np.inf
    assert np.isnan(got[2, 0]) and got[2, 1] == np.inf and got[2, 5] == np.inf
    for b in (0, 2, 3):
        assert np.isneginf(got[b, 6]) and np.isneginf(got[b, 7])  # the lowest value times 1.5 passes the type
        assert np.array_equal(got[b, 8:], x[b, 8:])


def test_process_counts_bias_and_bounds():
    """Counts past 2^16, all in one token; ids out of range in device lists count
    for nothing and a bias listed twice counts once, the last; mask rows out of
    range are no masks; spans."""
    import torch

    V, H = 9000, 70000
    x = torch.randn((3, V), device="cuda", dtype=torch.float64)
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    i64 = lambda a: torch.tensor(a, dtype=torch.int64, device="cuda")  # noqa: E731
    f64 = lambda a: torch.tensor(a, dtype=torch.float64, device="cuda")  # noqa: E731
    hist = torch.full((H + 4,), 8500, dtype=torch.int32, device="cuda")
    hist[H:] = i32([-1, V, 2**31 - 1, -2**31])
    spans = i64([0, H + 4, 5, 5, 100, 110])
    bias_ids, bias = i32([3, -1, 3, V, 8999, 3]), f64([1.0, 9.0, 2.0, 9.0, 0.25, 4.0])
    mask = torch.zeros((1, (V + 31) // 32), dtype=torch.int32, device="cuda")
    out = torch.empty_like(x)
    c = _native.default_context()
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    r, f, p, off = f64([1.0, 2.0, 1.0]), f64([0.5, 0.5, 0.25]), f64([0.25, 0.0, 0.0]), i64([0, 6, 6, 6])
    rows = i32([-1, 1, 0])
    c.process_logits(x.data_ptr(), _native.PLH_F64, V, 3, V, hist.data_ptr(), spans.data_ptr(), None, r.data_ptr(),
                     f.data_ptr(), p.data_ptr(), bias_ids.data_ptr(), bias.data_ptr(), off.data_ptr(), mask.data_ptr(),
                     mask.shape[1], 1, rows.data_ptr(), out.data_ptr(), V, _native.PLH_SAMPLE_HIST_SPANS)
    ref = x.clone()
    ref[0, 3] += 4.0
    ref[0, 8999] += 0.25
    ref[0, 8500] -= 0.5 * H + 0.25
    ref[2] = -torch.inf
    assert torch.equal(out, ref)


def test_process_streams_and_graph():
    """On a side stream, and captured into a graph whose replays, on inputs that
    change, match eager calls."""
    import torch

    V, B = 20000, 4
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.empty((B, V), device="cuda")
    hist = torch.randint(0, V, (B * 100,), generator=g, device="cuda").to(torch.int32)
    off = (100 * torch.arange(B + 1, device="cuda")).long()
    f = torch.full((B,), 0.5, dtype=torch.float64, device="cuda")
    mask = torch.randint(-2**31, 2**31 - 1, (B, V // 32), generator=g, device="cuda").to(torch.int32)
    out = torch.empty_like(x)
    c = _native.Context(0)

    def call(o):
        c.set_stream(torch.cuda.current_stream().cuda_stream)
        c.process_logits(x.data_ptr(), _native.PLH_F32, V, B, V, hist.data_ptr(), off.data_ptr(), None, None,
                         f.data_ptr(), None, None, None, None, mask.data_ptr(), V // 32, B, None, o.data_ptr(), V)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x.normal_(generator=g)
        call(out)
    s.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        call(out)
    for i in range(3):
        x.normal_(generator=g)
        eager = torch.empty_like(x)
        call(eager)
        torch.cuda.synchronize()
        out.fill_(0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
    c.close()


def test_process_refusals_of_the_library():
    import torch

    c = _native.Context(0)
    x = torch.zeros((4, 64), device="cuda")
    m = torch.zeros((4, 2), dtype=torch.int32, device="cuda")
    none = [None] * 9

    def go(ptr, code=0, ld=64, B=4, V=64, lists=none, mask=None, mask_ld=2, rows=4, row=None, o=x.data_ptr(), ldo=64,
           flags=0):
        c.process_logits(ptr, code, ld, B, V, *lists, mask, mask_ld, rows, row, o, ldo, flags)

    p = x.data_ptr()
    go(p)
    go(None, B=0)
    with pytest.raises(ValueError):
        go(None)
    with pytest.raises(ValueError):
        go(p, code=_native.PLH_BF16)
    with pytest.raises(ValueError):
        go(p, B=-1)
    with pytest.raises(ValueError):
        go(p, V=0)
    with pytest.raises(ValueError):
        go(p, ld=63)
    with pytest.raises(ValueError):
        go(p, o=p, ldo=65, B=3)
    with pytest.raises(ValueError):
        go(p, o=p + 16)  # rows that partly overlap
    with pytest.raises(ValueError):
        go(p + 1, B=1, V=32)
    with pytest.raises(ValueError):
        go(p, flags=1)
    with pytest.raises(ValueError):
        go(p, mask=m.data_ptr(), mask_ld=1)
    with pytest.raises(ValueError):
        go(p, mask=m.data_ptr(), rows=3)
    with pytest.raises(ValueError):
        go(p, lists=[None, p] + [None] * 7)  # hist_off without hist_ids
    with pytest.raises(ValueError):
        go(p, lists=[None] * 8 + [p])  # bias_off without bias
    go(p, B=4, V=32, o=p + 4 * 32)  # interleaved rows
    c.close()


# ------------------------------------------------------------ log probabilities


def _check_logprobs(res, x, ids, n):
    for b in range(x.shape[0]):
        ref = O.logprobs_row(x[b])
        order = O.order(x[b])
        err = O.logprobs_error(x[b]) if x.dtype == np.float32 and np.isfinite(ref).any() else 2.0 ** -40

        def near(got, want):
            want = np.asarray(want)
            assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(np.isinf(got), np.isinf(want))
            fin = np.isfinite(want)
            half = 2.0 ** -24 if x.dtype == np.float32 else 2.0 ** -50
            assert np.all(np.abs(got[fin] - want[fin]) <= err + half * np.abs(want[fin])), (b, got, want)

        if ids is not None:
            near(np.array([res.logprob[b]], np.float64), ref[[ids[b]]])
            assert res.rank[b] == 1 + int(np.flatnonzero(order == ids[b])[0])
        assert np.array_equal(res.top_ids[b], order[:n]), (b, res.top_ids[b], order[:n])
        near(res.top_logprobs[b].astype(np.float64), ref[order[:n]])


def _hard_rows(g, V, dt):
    """Rows that a selection goes wrong on."""
    x = g.normal(0, 3, (12, V))
    x[1] = 0.25                                    # one value
    x[2] = np.sort(x[2])                           # ascending
    x[3] = -np.sort(-x[3])                         # descending
    x[4] = -np.inf                                 # nothing
    x[5] = -np.inf
    x[5, g.integers(0, V, 3)] = 1.0                # few tokens allowed
    x[6] = np.round(x[6])                          # many ties
    x[7, g.random(V) < 0.9] = -np.inf
    x[8] = np.where(g.random(V) < 0.5, 0.0, -0.0)  # zeros of both signs
    x[9, V // 2] = np.nan
    x[9, V // 3] = np.inf
    x[10] *= 1e4                                   # far apart
    x[11] = np.finfo(dt).min
    x[11, V - 1] = 5.0                             # masks of the type's lowest value
    return x.astype(dt)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V", SIZES + [152064])
def test_logprobs_match_oracle(V, dt):
    g = np.random.default_rng(V)
    x = _hard_rows(g, V, dt)
    ids = g.integers(0, V, x.shape[0])
    for n in (0, 1, 5, 20, 64):
        if n <= V:
            print(f"[logprobs] V={V} {dt.__name__} n={n}", flush=True)
            _check_logprobs(token_logprobs(x, ids, n), x, ids, n)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V", [4000, 40000])
@pytest.mark.parametrize("B", [1, 600])  # several segments, and one of all chunks
def test_logprobs_many_nan_and_like_values(B, V, dt):
    """More NaNs, or more tokens of one value, than are asked for, in one chunk or
    another, or each chunk with larger values than the one before."""
    g = np.random.default_rng(V)
    x = g.normal(0, 1, (8, V))
    for b, at in enumerate([slice(0, 70), slice(V - 70, V), slice(V // 2, V // 2 + 64), slice(0, V, V // 65)]):
        x[b, at] = np.nan
    x[4, V // 2:] = 9.0
    x[5] = np.floor(np.arange(V) / 100)
    x[6, ::2] = 3.0
    x[7] = np.arange(V) // 4096 + g.random(V)
    x = x.astype(dt)
    for n in (1, 20, 64):
        print(f"[logprobs] like values B={B} V={V} {dt.__name__} n={n}", flush=True)
        res = token_logprobs(np.tile(x, (-(-B // 8), 1))[:max(B, 8)], None, n)
        _check_logprobs(type(res)(None, None, *(a[:8] for a in res[2:])), x, None, n)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,V", [(300, 20000), (2100, 8300), (1, 300000)])
def test_logprobs_row_shares(B, V, dt):
    """Batches whose rows are shared out differently over workgroups: several
    segments of one or more chunks, one segment of several chunks."""
    g = np.random.default_rng(B)
    x = np.tile(_hard_rows(g, V, dt), (-(-B // 12), 1))[:B]
    ids = g.integers(0, V, B)
    print(f"[logprobs] B={B} V={V} {dt.__name__}", flush=True)
    res = token_logprobs(x, ids, 20)
    some = np.unique(g.integers(0, B, 40))
    cut = type(res)(*(a[some] for a in res))
    _check_logprobs(cut, x[some], ids[some], 20)
    same = np.arange(B) % 12 == 4  # like rows, like answers
    assert (res.top_ids[same] == np.arange(20)).all()


def test_logprobs_torch_strides_ids_and_no_ids():
    import torch

    V, B = 12345, 5
    buf = torch.randn((B, V + 6), device="cuda")
    x = buf[:, 3:3 + V]
    host = x.cpu().numpy()
    ids = torch.tensor([0, V - 1, -1, V, 2**40], device="cuda")
    res = token_logprobs(x, ids, 7)
    assert res.logprob.is_cuda and res.rank.dtype == torch.int32 and res.top_logprobs.shape == (B, 7)
    lp, rank = res.logprob.cpu().numpy(), res.rank.cpu().numpy()
    assert np.isnan(lp[2:]).all() and not rank[2:].any()
    _check_logprobs(type(res)(lp[:2], rank[:2], *(t.cpu().numpy()[:2] for t in res[2:])), host[:2], [0, V - 1], 7)
    alone = token_logprobs(x, None, 7)
    assert alone.logprob is None and torch.equal(alone.top_ids, res.top_ids)
    assert token_logprobs(x[:0], ids[:0], 3).top_ids.shape == (0, 3)
    with pytest.raises(TypeError):
        token_logprobs(x.half(), ids)
    with pytest.raises(ValueError):
        token_logprobs(buf.T, None, 1)
    with pytest.raises(TypeError):
        token_logprobs(x, ids.float())


def test_logprobs_streams_workspace_and_graphs():
    """Calls of one context on two streams, with nothing between them; two
    graphs captured from one context (captured calls use no workspace), replayed
    at once on two streams, match eager calls."""
    import torch

    V, B, n = 100000, 3, 20
    c = _native.Context(0)
    xs = [torch.randn((B, V), device="cuda") for _ in range(2)]
    ids = torch.tensor([5, 7, 9], dtype=torch.int32, device="cuda")
    new = lambda: [torch.empty(B, device="cuda"), torch.empty_like(ids),  # noqa: E731
                   torch.empty((B, n), dtype=torch.int32, device="cuda"), torch.empty((B, n), device="cuda")]

    def call(x, o):
        c.set_stream(torch.cuda.current_stream().cuda_stream)
        c.logprobs(x.data_ptr(), _native.PLH_F32, V, B, V, ids.data_ptr(), o[0].data_ptr(), o[1].data_ptr(), n,
                   o[2].data_ptr(), o[3].data_ptr())

    want = [new(), new()]
    for x, o in zip(xs, want):
        call(x, o)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [new(), new()]
    for _ in range(3):
        for s, x, o in zip(streams, xs, got):
            with torch.cuda.stream(s):
                call(x, o)
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))
    graphs = []
    got = [new(), new()]
    for s, x, o in zip(streams, xs, got):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call(x, o)
        graphs.append(g)
    for i in range(3):
        for x, o in zip(xs, got):
            x.normal_()
            [t.zero_() for t in o]
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for x, o, w in zip(xs, got, want):
            call(x, w)
            torch.cuda.synchronize()
            assert torch.equal(o[1], w[1]) and torch.equal(o[2], w[2])
            # the graph's one segment adds in another order
            assert float((o[0] - w[0]).abs().max()) < 1e-5 and float((o[3] - w[3]).abs().max()) < 1e-5
    c.set_stream(None)
    c.close()


def test_logprobs_refusals_of_the_library():
    import torch

    c = _native.Context(0)
    x = torch.zeros((2, 100), device="cuda")
    i = torch.zeros(200, dtype=torch.int32, device="cuda")
    p, q = x.data_ptr(), i.data_ptr()
    for args in [
        (None, 0, 100, 2, 100, q, p, q),
        (p, 2, 100, 2, 100, q, p, q),
        (p, 0, 99, 2, 100, q, p, q),
        (p, 0, 100, -1, 100, q, p, q),
        (p, 0, 100, 2, 0, q, p, q),
        (p, 0, 100, 2, 100, q, None, q),
        (p, 0, 100, 2, 100, q, p, None),
        (p, 0, 100, 2, 100, q, p, q, 65, q, p),
        (p, 0, 100, 2, 100, q, p, q, -1, q, p),
        (p, 0, 100, 2, 5, q, p, q, 6, q, p),
        (p, 0, 100, 2, 100, q, p, q, 5, None, p),
        (p, 0, 100, 2, 100, q, p, q, 5, q, None),
        (p + 2, 0, 100, 1, 90, q, p, q),
    ]:
        with pytest.raises(ValueError):
            c.logprobs(*args)
    c.logprobs(None, 0, 100, 0, 100, None, None, None)
    c.logprobs(p, 0, 100, 2, 100, None, None, None)
    c.close()


def test_offsets_past_32_bits_and_very_many_rows():
    """More than 2^31 logits in more rows than a grid's y holds: the last rows."""
    import torch

    B, V = 70001, 31000
    print("[logits] 70001 x 31000", flush=True)
    x = torch.zeros((B, V), device="cuda")
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    rows = torch.tensor([0, 65535, 65536, 69273, B - 1], device="cuda")  # 69273 * 31000 passes 2^31
    x[rows] = torch.randn((5, V), generator=g, device="cuda")
    host = x[rows].cpu().numpy()
    ids = torch.zeros(B, dtype=torch.int32, device="cuda")
    ids[rows] = 77
    res = token_logprobs(x, ids, 3)
    cut = type(res)(*(t[rows].cpu().numpy() for t in res))
    _check_logprobs(cut, host, np.full(5, 77), 3)
    assert bool((res.top_ids[1:65535] == torch.arange(3, device="cuda")).all())  # rows of zeros
    words = torch.from_numpy(pack_mask(np.arange(V) % 3 == 0, V).view(np.int32)).cuda()[None]
    mask_row = torch.full((B,), -1, dtype=torch.int32, device="cuda")
    mask_row[rows] = 0
    f = torch.full((B,), 0.5, dtype=torch.float64, device="cuda")
    hist = torch.tensor([3, 3, 6], dtype=torch.int32, device="cuda")
    spans = torch.tensor([0, 3], device="cuda").repeat(B)
    c = _native.default_context()
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    c.process_logits(x.data_ptr(), _native.PLH_F32, V, B, V, hist.data_ptr(), spans.data_ptr(), None, None, f.data_ptr(),
                     None, None, None, None, words.data_ptr(), words.shape[1], 1, mask_row.data_ptr(), x.data_ptr(), V,
                     _native.PLH_SAMPLE_HIST_SPANS)
    want = host.astype(np.float64)
    want[:, 3] -= 1.0
    want[:, 6] -= 0.5
    want = want.astype(np.float32)
    want[:, np.arange(V) % 3 != 0] = -np.inf
    assert np.array_equal(x[rows].cpu().numpy(), want)
    zero = x[1000]
    assert float(zero[3]) == -1.0 and float(zero[6]) == -0.5 and float(zero.sum()) == -1.5


@pytest.mark.parametrize("dt", DTYPES)
def test_token_logits(dt):
    """The chosen tokens' logits, NaN for ids outside the vocabulary; rows of a wider
    buffer; refusals."""
    import torch

    B, V, ld = 300, 1001, 1010
    x = torch.randn((B, ld), device="cuda", dtype=getattr(torch, np.dtype(dt).name))
    ids = torch.randint(0, V, (B,), device="cuda").to(torch.int32)
    ids[[0, 1, 299]] = torch.tensor([-1, V, V - 1], dtype=torch.int32, device="cuda")
    out = torch.zeros(B + 1, device="cuda", dtype=x.dtype)
    code = _native.dtype_code(dt)
    c = _native.Context(0)
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    p, i, o = x.data_ptr(), ids.data_ptr(), out.data_ptr()
    c.token_logits(p, code, ld, B, V, i, o)
    got = out.cpu().numpy()
    assert np.isnan(got[:2]).all() and got[B] == 0
    assert np.array_equal(got[2:B], x.gather(1, ids.long().clamp(0, V - 1)[:, None])[2:, 0].cpu().numpy())
    c.token_logits(None, code, ld, 0, V, None, None)
    for args in [(None, code, ld, B, V, i, o), (p, code, ld, B, V, None, o), (p, code, ld, B, V, i, None),
                 (p, 2, ld, B, V, i, o), (p, code, V - 1, B, V, i, o), (p, code, ld, -1, V, i, o),
                 (p, code, ld, B, 0, i, o), (p + 2, code, ld, 1, V, i, o), (p, code, ld, B, V, i, o + 2)]:
        with pytest.raises(ValueError):
            c.token_logits(*args)
    c.close()


def test_calls_on_cuda_tensors_wait_for_nothing():
    """Calls with host rules, masks and ids return while their logits' producer runs,
    and many of them in flight keep their own arguments."""
    import torch

    V, B = 5000, 4
    g = np.random.default_rng(11)
    a = torch.randn((8192, 8192), device="cuda", dtype=torch.bfloat16)
    b = torch.empty_like(a)
    src = torch.randn((B, V), device="cuda")
    x = torch.zeros_like(src)
    hosts = [(LogitRules(0.5, 0.25, {int(t): float(v) for t, v in zip(g.integers(0, V, 9), g.normal(0, 2, 9))}),
              [g.integers(0, V, 30).tolist() for _ in range(B)], pack_mask(g.random(V) < 0.5, V)[None],
              g.integers(0, V, B)) for _ in range(16)]

    def calls():
        got = []
        for rule, hist, mask, ids in hosts:
            y = process_logits(x, rule, contexts=hist, masks=mask, mask_rows=[0] * B)
            got.append((y, token_logprobs(x, ids, 5)))
        return got

    def produce():
        for _ in range(60):  # tens of milliseconds
            torch.mm(a, a, out=b)
        x.copy_(src)
        e = torch.cuda.Event()
        e.record()
        return e

    produce()
    calls()  # the allocators' first time
    torch.cuda.synchronize()
    x.zero_()
    done = produce()
    got = calls()
    assert not done.query(), "a call waited for the logits' producer"
    torch.cuda.synchronize()
    host = src.cpu().numpy()
    for (rule, hist, mask, ids), (y, lp) in zip(hosts, got):
        rows = [(1.0, rule, 30, 0, None)] * B
        _check(y.cpu().numpy(), host, rows, [np.asarray(h) for h in hist], [mask[0]] * B)
        _check_logprobs(type(lp)(*(t.cpu().numpy() for t in lp)), host, ids, 5)
    assert token_logprobs(x[:0], [], 3).rank.shape == (0,)


def test_calls_under_capture():
    """Calls whose arguments are all on the device are captured; host arguments are
    refused, and the capture goes on."""
    import torch

    V, B = 5000, 4
    x = torch.randn((B, V), device="cuda")
    masks = torch.randint(-2**31, 2**31 - 1, (B, -(-V // 32)), device="cuda").to(torch.int32)
    ids = torch.tensor([1, 2, 3, 4], dtype=torch.int32, device="cuda")
    process_logits(x, masks=masks)
    token_logprobs(x, ids, 5)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            process_logits(x, LogitRules(logit_bias={3: 1.0}))
        with pytest.raises(RuntimeError, match="captured"):
            token_logprobs(x, [1, 2, 3, 4])
        y = process_logits(x, masks=masks)
        plain = process_logits(x, LogitRules(), SamplingParams(), [[1, 2]] * B)
        lp = token_logprobs(x, ids, 5)
    for i in range(3):
        x.normal_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, process_logits(x, masks=masks)) and torch.equal(plain, x)
        _check_logprobs(type(lp)(*(t.cpu().numpy() for t in lp)), x.cpu().numpy(), ids.cpu().numpy(), 5)
    _native.default_context().set_stream(None)


def test_the_longest_row():
    """V = 2^31 - 1, the most that the entry points take: the last chunk's bounds."""
    import torch

    V = 2**31 - 1
    print("[logits] one row of 2^31 - 1", flush=True)
    x = torch.zeros((1, V), device="cuda")
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    at = [0, 4095, 4096, V - 4096, V - 2, V - 1]
    bias_ids, bias = i32(at), torch.arange(1.0, 7.0, dtype=torch.float64, device="cuda")
    hist, off = i32([V - 1, 5, V - 1]), torch.tensor([0, 3], device="cuda")
    f = torch.full((1,), 0.25, dtype=torch.float64, device="cuda")
    b_off = torch.tensor([0, 6], device="cuda")
    mask = torch.full((1, (V + 31) // 32), -1, dtype=torch.int32, device="cuda")
    mask[0, -1] = 0x7FFFFFFF & ~(1 << 29)  # token V - 2
    out = torch.full((1, V + 1), 7.0, device="cuda")  # and nothing past the row
    c = _native.default_context()
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    for o in (out, x):  # out of place, then in place
        c.process_logits(x.data_ptr(), _native.PLH_F32, V, 1, V, hist.data_ptr(), off.data_ptr(), None, None, f.data_ptr(),
                         None, bias_ids.data_ptr(), bias.data_ptr(), b_off.data_ptr(), mask.data_ptr(), mask.shape[1], 1,
                         None, o.data_ptr(), V)
        y = o[0, :V]
        assert y[at].tolist() == [1.0, 2.0, 3.0, 4.0, -np.inf, 5.5] and float(y[5]) == -0.25
        assert int((y != 0).sum()) == 7
    assert float(out[0, V]) == 7.0
    del out
    res = token_logprobs(x, torch.tensor([V - 1], device="cuda"), 5)
    assert res.top_ids.tolist() == [[V - 1, V - 4096, 4096, 4095, 0]] and res.rank.tolist() == [1]
    e = np.exp(np.array([5.5, 4.0, 3.0, 2.0, 1.0, -0.25]))
    lse = np.log(e.sum() + V - 7)
    # the float32 terms (2^-23 of each), their float64 sum and one rounding
    assert np.allclose(res.top_logprobs.cpu().numpy()[0], np.array([5.5, 4, 3, 2, 1]) - lse, rtol=2.0 ** -24, atol=2.0 ** -22)


def test_sizes_past_int32_are_refused():
    """Not taken modulo 2^32 (nothing but the allocation happens at these sizes)."""
    import torch

    print("[logits] 2^32 + 10 tokens", flush=True)
    x = torch.empty(2**32 + 10, device="cuda")
    for t in (x[None], x[:, None]):
        with pytest.raises(ValueError, match="2\\^31"):
            process_logits(t, out=t)
        with pytest.raises(ValueError, match="2\\^31"):
            token_logprobs(t, None, 1)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("V", [4063, 4064, 4095, 4096, 4097, 4100, 8191, 8195, 12287, 12289])
def test_process_around_its_chunks(V, dt):
    """k_process takes 4096 tokens a workgroup: rows that end just before, at and behind
    a chunk, in place and not."""
    import torch

    print(f"[process] chunks V={V} {dt.__name__}", flush=True)
    x, rows, hist, masks = _case(V, 7, V, dt)
    got = _run_numpy(x, rows, hist, masks)
    _check(got, x, rows, hist, masks)
    t = torch.from_numpy(x).cuda()
    words = np.stack([m if m is not None else pack_mask(np.ones(V, bool), V) for m in masks])
    process_logits(t, [k[1] for k in rows], [SamplingParams(repetition_penalty=k[0]) for k in rows], hist,
                   prompt_lens=[k[3] for k in rows], masks=words, out=t)
    assert np.array_equal(t.cpu().numpy(), got)


def _shares(B, V, dt, cus):
    """(segments, chunks of one) of rows: at most two workgroups a CU, whole chunks of
    8192 float32 or 4096 float64 tokens each, one segment up to three chunks."""
    chunks = -(-V // (8192 if dt == np.float32 else 4096))
    each = chunks if chunks <= 3 else min(chunks, -(-B * chunks // (2 * cus)))
    return -(-chunks // each), each


@pytest.mark.parametrize("n", [0, 20, 64])
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("B,V", [(256, 128256), (200, 70000), (100, 152064), (140, 41000), (190, 41000)])
def test_logprobs_segments_of_many_chunks(B, V, dt, n):
    """Rows cut into several segments of several chunks each: a segment's own threshold
    from its third chunk on, away from the row's start, and the second launch's join."""
    import torch

    cus = torch.cuda.get_device_properties(0).multi_processor_count
    segs, each = _shares(B, V, dt, cus)
    assert segs >= 2 and each >= (2 if B == 140 else 3), (segs, each)  # 140 float32 rows: segments of two
    g = np.random.default_rng(V + n)
    kinds = np.concatenate([_hard_rows(g, V, dt), np.zeros((8, V), dt)])
    more = kinds[12:]
    more[:] = g.normal(0, 1, more.shape)
    for b, at in enumerate([slice(0, 70), slice(V - 70, V), slice(V // 2, V // 2 + 64), slice(0, V, V // 65)]):
        more[b, at] = np.nan
    more[4, V // 2:] = 9.0                       # like values over whole segments
    more[5] = np.floor(np.arange(V) / 100)       # every chunk larger than the one before
    more[6, ::2] = 3.0
    more[7] = np.arange(V)[::-1] // 4096 + g.random(V)  # the best at each segment's start
    rows = np.arange(B) % 20
    ids = g.integers(0, V, B)
    print(f"[logprobs] segments B={B} V={V} {dt.__name__} n={n}: {segs} of {each} chunks", flush=True)
    res = token_logprobs(torch.from_numpy(kinds).cuda()[torch.from_numpy(rows).cuda()], ids, n)
    res = type(res)(*(t.cpu().numpy() for t in res))
    _check_logprobs(type(res)(*(a[B - 20:] for a in res)), kinds[rows[B - 20:]], ids[B - 20:], n)
    # like rows, like answers
    for k in range(20):
        same = res.top_ids[rows == k]
        assert (same == same[0]).all()


def test_staged_copies():
    """Memory that is given out twice is two buffers, and is not given again before its
    copy has ended; refusals leave it given."""
    import torch

    c = _native.Context(0)
    n = 100_000
    d = torch.zeros((40, n), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    a = torch.randn((4096, 4096), device="cuda")
    for stream in (None, side):
        with torch.cuda.stream(stream):
            torch.cuda.synchronize()
            for _ in range(20):
                torch.mm(a, a)
            c.set_stream(torch.cuda.current_stream().cuda_stream)
            for i in range(40):
                s = c.stage(n - i)
                s[:] = i + 1
                c.stage_h2d(d[i].data_ptr(), s)
            got = d.clone()
        torch.cuda.synchronize()
        for i in range(40):
            assert bool((got[i, :n - i] == i + 1).all()) and not bool(got[i, n - i:].any())
        d.zero_()
    s, t = c.stage(10), c.stage(10)
    assert s.ctypes.data != t.ctypes.data
    with pytest.raises(ValueError):
        c.stage_h2d(d.data_ptr(), np.zeros(10, np.uint8))
    with pytest.raises(ValueError):
        c.stage_h2d(None, s)
    with pytest.raises(ValueError):
        c._check(c.lib.plh_stage_h2d(c.handle, d.data_ptr(), s.ctypes.data, 1 << 30))
    c.stage_h2d(None, s[:0])  # given back alone
    with pytest.raises(ValueError):
        c.stage_h2d(d.data_ptr(), s)
    c.close()
