"""The way from hidden states to an answer, as a serving loop runs it: e4m3
logits, rules and grammar masks, sampling, log probabilities, through
``BatchSampler`` with histories on the device (needs an MI355X)."""

from __future__ import annotations

import numpy as np
import pytest

import oracle
from oracle import logits as O
from pagellm_amd.engine import BatchSampler, DeviceHistories
from pagellm_amd.fp8 import Fp8LogitsHead
from pagellm_amd.logits import LogitRules, pack_mask, process_logits
from pagellm_amd.params import SamplingParams, make_rng

pytestmark = pytest.mark.gpu

V, D = 3000, 256
ROWS = [  # (params, rules, prompt length, under a grammar)
    (SamplingParams(temperature=0.0), None, 5, False),
    (SamplingParams(temperature=0.0, repetition_penalty=1.3), LogitRules(0.4, 0.2), 9, False),
    (SamplingParams(temperature=0.8, top_k=20), LogitRules(logit_bias={7: 12.0, 8: -np.inf}), 7, True),
    (SamplingParams(temperature=1.0, top_p=0.9, repetition_penalty=1.2), None, 12, True),
    (SamplingParams(temperature=0.0), LogitRules(0.0, 3.0), 3, True),
]


@pytest.mark.parametrize("on_gpu", [True, False])
def test_steps_match_the_oracle(on_gpu):
    g = np.random.default_rng(3)
    norm = (1 + 0.1 * g.standard_normal(D)).astype(np.float32)
    head = Fp8LogitsHead(norm, (0.1 * g.standard_normal((D, V))).astype(np.float32))
    hist = DeviceHistories(V, max_seqs=8, max_len=64)
    sampler = BatchSampler(hist)
    keys = list("abcde")
    tokens = {k: [int(t) for t in g.integers(0, V, row[2])] for k, row in zip(keys, ROWS)}
    for k in keys:
        hist.add(k, tokens[k])
    rngs, ref_rngs = ([make_rng(i, 0) for i in range(5)] for _ in range(2))
    for step in range(6):
        logits = head(g.standard_normal((5, D)).astype(np.float32))
        x = logits.cpu().numpy()
        masks = np.stack([pack_mask(g.random(V) < 0.3, V), pack_mask([5, 7, 8, 11], V)])
        at = [None, None, 1, 0, 1 if step % 2 else 0]
        ids, lps = sampler.sample(logits if on_gpu else x, [r[0] for r in ROWS], rngs, keys, rules=[r[1] for r in ROWS],
                                  masks=masks, mask_rows=at, logprobs=5)
        assert np.array_equal(logits.cpu().numpy(), x)  # the caller's logits stay as they were
        for b, (k, (params, rule, plen, _)) in enumerate(zip(keys, ROWS)):
            rule = rule or LogitRules()
            ruled = not rule.neutral
            y = O.process_row(x[b], history=tokens[k], out_start=plen, rep=params.repetition_penalty if ruled else 1.0,
                              freq=rule.frequency_penalty, pres=rule.presence_penalty,
                              bias=list(rule.logit_bias.items()), mask=masks[at[b]] if at[b] is not None else None)
            y = y.astype(np.float32)
            rest = SamplingParams(temperature=params.temperature, top_k=params.top_k, top_p=params.top_p,
                                  repetition_penalty=1.0 if ruled else params.repetition_penalty)
            u = None if params.greedy else ref_rngs[b].random()
            want = oracle.sample(y, rest, u, tokens[k])
            assert ids[b] == want, (step, k)
            order = O.order(x[b])
            assert lps.rank[b] == 1 + int(np.flatnonzero(order == want)[0])
            assert np.array_equal(lps.top_ids[b], order[:5])
            lp = O.logprobs_row(x[b])
            tol = O.logprobs_error(x[b]) + 2.0 ** -24 * 50
            assert abs(lps.logprob[b] - lp[want]) <= tol
            assert np.all(np.abs(lps.top_logprobs[b] - lp[order[:5]]) <= tol)
            tokens[k].append(int(want))
            assert np.array_equal(hist.download(k), tokens[k])
    for a, b in zip(rngs, ref_rngs):
        assert a.random() == b.random()


def test_rows_without_rules_keep_their_ids_and_errors_change_nothing():
    import torch

    g = np.random.default_rng(0)
    x = g.normal(0, 2, (2, V)).astype(np.float32)
    params = SamplingParams(temperature=1.0, repetition_penalty=1.2, top_p=0.9)
    ids = []
    for rules in (None, [None, LogitRules(0.5)]):
        hist = DeviceHistories(V, max_seqs=2, max_len=8)
        hist.add(0, [1, 2, 3], prompt_len=1)
        hist.add(1, [4, 5, 6])
        sampler = BatchSampler(hist)
        rngs = [make_rng(1, 0), make_rng(2, 0)]
        with pytest.raises(IndexError):
            sampler.sample(x, params, rngs, [0, 1], rules=LogitRules(logit_bias={V: 1.0}))
        with pytest.raises(ValueError):
            sampler.sample(x, params, rngs, [0, 1], masks=np.zeros((1, 94), np.uint32))
        with pytest.raises(ValueError):
            sampler.sample(x, params, rngs, [0, 1], logprobs=65)
        with pytest.raises(TypeError):  # masks on torch's stream, logits on the context's
            sampler.sample(x, params, rngs, [0, 1], masks=torch.zeros((2, 94), dtype=torch.int32, device="cuda"))
        ids.append(sampler.sample(x, params, rngs, [0, 1], rules=rules))
        assert list(hist.output_starts([0, 1])) == [1, 3]
    assert ids[0][0] == ids[1][0]
    with pytest.raises(ValueError):
        hist.remove(0)
        hist.add(0, [1, 2], prompt_len=3)
    assert sampler.sample(x[:0], [], [], [], logprobs=2)[1].top_ids.shape == (0, 2)


@pytest.mark.parametrize("dt", [np.float32, np.float64])
@pytest.mark.parametrize("on_gpu", [True, False])
@pytest.mark.parametrize("n", [65, 3000, 50257])
def test_rows_of_which_rules_and_masks_leave_nothing(n, on_gpu, dt):
    """Such a row gives -1, joins nothing and has no log probability, greedy or
    sampled, whatever rows stand beside it; its sequence goes on in a later step."""
    import torch

    print(f"[answer] nothing left V={n} {dt.__name__} on_gpu={on_gpu}", flush=True)
    g = np.random.default_rng(n)
    x = g.normal(0, 2, (8, n)).astype(dt)
    x[7] = -np.inf  # the model's own: no rule and no mask of this row's did it
    greedy, drawn = SamplingParams(temperature=0.0, repetition_penalty=1.3), SamplingParams(temperature=0.9, top_p=0.9)
    params = [greedy, drawn, drawn, greedy, drawn, drawn, greedy, greedy]
    rules = [None] * 8
    rules[3] = LogitRules(logit_bias={7: -np.inf, 9: -np.inf})  # all that the mask allows
    rules[6] = LogitRules(0.5, 0.1)
    masks = np.zeros((4, (n + 31) // 32), dtype=np.uint32)
    masks[1] = pack_mask([7, 9], n)
    masks[2] = pack_mask([3, 7, 9], n)
    masks[3, -1] = (0xFFFFFFFF << (n % 32)) & 0xFFFFFFFF if n % 32 else 0  # bits past the vocabulary
    at = [0, 0, 2, 1, None, 3, None, None]
    hist = DeviceHistories(n, max_seqs=8, max_len=16)
    sampler = BatchSampler(hist)
    keys = list("abcdefgh")
    tokens = {k: [3, 7, 9, b] for b, k in enumerate(keys)}
    for k in keys:
        hist.add(k, tokens[k], prompt_len=2)
    rngs, ref_rngs = ([make_rng(i, 0) for i in range(8)] for _ in range(2))
    logits = torch.from_numpy(x).cuda() if on_gpu else x
    words = torch.from_numpy(masks.view(np.int32)).cuda() if on_gpu else masks
    for given_masks in (words, None):  # a step under the masks, and one without
        ids, lps = sampler.sample(logits, params, rngs, keys, rules=rules if given_masks is not None else None,
                                  masks=given_masks, mask_rows=at if given_masks is not None else None, logprobs=3)
        for b, k in enumerate(keys):
            rule = rules[b] if given_masks is not None and rules[b] is not None else LogitRules()
            mask = masks[at[b]] if given_masks is not None and at[b] is not None else None
            rep = params[b].repetition_penalty
            y = O.process_row(x[b], history=tokens[k], out_start=2, rep=1.0 if rule.neutral else rep,
                              freq=rule.frequency_penalty, pres=rule.presence_penalty,
                              bias=list(rule.logit_bias.items()), mask=mask).astype(dt)
            rest = SamplingParams(temperature=params[b].temperature, top_p=params[b].top_p,
                                  repetition_penalty=rep if rule.neutral else 1.0)
            u = None if params[b].greedy else ref_rngs[b].random()  # drawn whether or not something is left
            order = O.order(x[b])
            assert np.array_equal(lps.top_ids[b], order[:3])
            if given_masks is not None and b in (0, 1, 3, 5):
                assert ids[b] == -1 and np.isnan(lps.logprob[b]) and lps.rank[b] == 0
            else:
                want = oracle.sample(y, rest, u, tokens[k])
                assert ids[b] == want, (b, ids[b], want)
                assert lps.rank[b] == 1 + int(np.flatnonzero(order == want)[0])
                tokens[k].append(int(want))
            assert hist.length(k) == len(tokens[k])
            assert np.array_equal(hist.download(k), tokens[k])
    for a, b in zip(rngs, ref_rngs):
        assert a.random() == b.random()


def test_masks_whose_rows_overlap_are_refused_before_a_generator_moves():
    import torch

    x = torch.randn((3, V), device="cuda")
    hist = DeviceHistories(V, max_seqs=3, max_len=8)
    for k in range(3):
        hist.add(k, [1, 2])
    rngs = [make_rng(k, 0) for k in range(3)]
    words = torch.from_numpy(pack_mask([4, 5], V).view(np.int32)).cuda()
    sampler = BatchSampler(hist)
    for masks in (words[None].expand(3, -1), torch.zeros(94 * 3, dtype=torch.int32, device="cuda").as_strided((3, 94), (93, 1))):
        with pytest.raises(ValueError, match="overlap"):
            sampler.sample(x, SamplingParams(), rngs, [0, 1, 2], masks=masks)
        with pytest.raises(ValueError, match="overlap"):
            process_logits(x, masks=masks)
    assert [r.random() for r in rngs] == [make_rng(k, 0).random() for k in range(3)]
    # what is meant: one row of masks for all
    ids = sampler.sample(x, SamplingParams(), rngs, [0, 1, 2], masks=words[None].expand(1, -1), mask_rows=[0, 0, 0])
    assert set(ids) <= {4, 5}


def test_the_chain_captured_behind_eager_calls():
    """e4m3 logits, masks and log probabilities in one graph, captured while the context's
    workspace is in use by eager calls of the default stream; replays between such calls
    match them."""
    import torch

    from pagellm_amd.logits import token_logprobs

    n, rows = 100000, 3
    g = np.random.default_rng(2)
    norm = np.ones(D, np.float32)
    head = Fp8LogitsHead(norm, (0.1 * g.standard_normal((D, n))).astype(np.float32))
    h = torch.randn((rows, D), device="cuda")
    masks = torch.from_numpy(np.stack([pack_mask(g.random(n) < 0.4, n) for _ in range(rows)]).view(np.int32)).cuda()
    ids = torch.tensor([5, 6, 7], dtype=torch.int32, device="cuda")

    def chain():
        logits = head(h)
        left = process_logits(logits, masks=masks)
        return logits, left, token_logprobs(left, ids, 20)

    chain()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        chain()
    torch.cuda.synchronize()
    chain()  # several workgroups a row: the workspace
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = chain()
    for _ in range(3):
        h.normal_()
        want = chain()
        graph.replay()
        again = chain()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(again[1], want[1])
        assert torch.equal(got[2].top_ids, want[2].top_ids) and torch.equal(got[2].rank, want[2].rank)
        assert torch.equal(again[2].top_logprobs, want[2].top_logprobs)
        # one segment a row in the graph: another order of float64 sums, one rounding
        fin = torch.isfinite(want[2].logprob)
        assert torch.equal(fin, torch.isfinite(got[2].logprob))
        assert float((got[2].top_logprobs - want[2].top_logprobs).abs().max()) < 2e-6
        assert float((got[2].logprob - want[2].logprob)[fin].abs().sum()) < 6e-6
