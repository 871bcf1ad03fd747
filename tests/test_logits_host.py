"""Host side of logits processing, log probabilities and e4m3 products: packing
and refusals that need no GPU."""

from __future__ import annotations

import math
from types import SimpleNamespace

import numpy as np
import pytest

from oracle import logits as O
from pagellm_amd import _native
from pagellm_amd.logits import LogitRules, _pack, _pack_rules, pack_mask, process_logits, token_logprobs

NO_GPU = SimpleNamespace(device=0)  # a context that no refused call reaches


def test_rules_validate_and_pack():
    with pytest.raises(ValueError):
        LogitRules(frequency_penalty=math.nan)
    with pytest.raises(ValueError):
        LogitRules(presence_penalty=math.inf)
    with pytest.raises(ValueError):
        LogitRules(logit_bias={3: math.nan})
    with pytest.raises(ValueError):
        LogitRules(logit_bias={3: math.inf})
    with pytest.raises(ValueError):
        LogitRules(logit_bias={-1: 1.0})
    with pytest.raises(ValueError):
        LogitRules(logit_bias={2**31: 1.0})
    assert LogitRules().neutral and not LogitRules(logit_bias={0: 0.0}).neutral
    assert LogitRules(presence_penalty=-1.0).penalises
    rules = [LogitRules(), LogitRules(0.5, 0.25, {7: 1.5, 2: -math.inf}), LogitRules(logit_bias={"4": 2})]
    f, p, ids, bias, off = _pack_rules(rules, 8)
    assert list(f) == [0, 0.5, 0] and list(p) == [0, 0.25, 0]
    assert list(ids) == [7, 2, 4] and list(bias) == [1.5, -math.inf, 2.0] and list(off) == [0, 0, 2, 3]
    with pytest.raises(IndexError):
        _pack_rules(rules, 7)
    assert _pack_rules([LogitRules()], 8)[2:] == (None, None, None)
    assert hash(rules[1]) == hash(LogitRules(0.5, 0.25)) and rules[1] != LogitRules(0.5, 0.25)
    # a dict given stays the caller's
    d = {1: 1.0}
    r = LogitRules(logit_bias=d)
    d[2] = 3.0
    assert r.logit_bias == {1: 1.0}


@pytest.mark.parametrize("V", [1, 31, 32, 33, 65, 1000])
def test_masks_pack(V):
    g = np.random.default_rng(V)
    ids = np.unique(g.integers(0, V, V // 2 + 1))
    words = pack_mask(ids, V)
    assert words.dtype == np.uint32 and words.shape == ((V + 31) // 32,)
    assert np.array_equal(np.flatnonzero(O.allowed(words, V)), ids)
    flags = np.zeros(V, dtype=bool)
    flags[ids] = True
    assert np.array_equal(pack_mask(flags, V), words)
    assert np.array_equal(pack_mask([int(t) for t in ids], V), words)
    assert not pack_mask([], V).any()
    with pytest.raises(IndexError):
        pack_mask([V], V)
    with pytest.raises(ValueError):
        pack_mask(np.zeros(V + 1, dtype=bool), V)


def test_pack_aligns_its_parts():
    parts = [np.arange(3, dtype=np.int32), None, np.arange(5, dtype=np.float64), np.zeros(0)]
    buf, offs = _pack(parts)
    assert offs[1] is None and all(o % 16 == 0 for o in offs if o is not None)
    assert np.array_equal(buf[offs[2]:offs[2] + 40].view(np.float64), parts[2])


def test_refusals_of_process_logits():
    x = np.zeros((2, 10), dtype=np.float32)
    go = lambda *a, **k: process_logits(*a, ctx=NO_GPU, **k)  # noqa: E731
    with pytest.raises(ValueError):
        go(x[0])
    with pytest.raises(ValueError):
        go(np.zeros((2, 0), dtype=np.float32))
    with pytest.raises(ValueError):
        go(x, [LogitRules()])
    with pytest.raises(IndexError):
        go(x, LogitRules(logit_bias={10: 1.0}))
    with pytest.raises(ValueError):
        go(x, contexts=[[1]])
    with pytest.raises(IndexError):
        go(x, LogitRules(0.1), contexts=[[1], [10]])
    with pytest.raises(ValueError):
        go(x, prompt_lens=[1, 1])
    with pytest.raises(ValueError):
        go(x, LogitRules(0.1), contexts=[[1], [2]], prompt_lens=[1])
    with pytest.raises(ValueError):
        go(x, LogitRules(0.1), contexts=[[1], [2]], prompt_lens=[1, -1])
    with pytest.raises(ValueError):
        go(x, masks=np.zeros((1, 1), np.uint32))  # one mask row for two rows
    with pytest.raises(ValueError):
        go(x, masks=np.zeros((2, 0), np.uint32))
    with pytest.raises(TypeError):
        go(x, masks=np.zeros((2, 1), np.int64))
    with pytest.raises(ValueError):
        go(x, masks=np.zeros(2, np.uint32)[None, :, None])
    with pytest.raises(IndexError):
        go(x, masks=np.zeros((1, 1), np.uint32), mask_rows=[0, 1])
    with pytest.raises(IndexError):
        go(x, masks=np.zeros((1, 1), np.uint32), mask_rows=[0, -2])
    with pytest.raises(ValueError):
        go(x, masks=np.zeros((1, 1), np.uint32), mask_rows=[0])
    with pytest.raises(ValueError):
        go(x, mask_rows=[0, 0])
    with pytest.raises(ValueError):
        go(x, out=x)


def test_refusals_of_token_logprobs():
    x = np.zeros((2, 10), dtype=np.float32)
    go = lambda *a, **k: token_logprobs(*a, ctx=NO_GPU, **k)  # noqa: E731
    with pytest.raises(ValueError):
        go(x[0])
    with pytest.raises(ValueError):
        go(np.zeros((2, 0), dtype=np.float32))
    for n in (-1, 11):
        with pytest.raises(ValueError):
            go(x, n_top=n)
    with pytest.raises(ValueError):
        go(np.zeros((2, 100), dtype=np.float32), n_top=65)
    with pytest.raises(ValueError):
        go(x, [1])
    for t in (-1, 10):
        with pytest.raises(IndexError):
            go(x, [0, t])


def test_null_contexts_and_sizes():
    lib = _native.load_library()
    assert lib.plh_process_logits(None, None, 0, 1, 1, 1, *[None] * 10, 1, 1, None, None, 1, 0) == -1
    assert lib.plh_logprobs(None, None, 0, 1, 1, 1, None, None, None, 0, None, None) == -1
    assert lib.plh_fp8_pack(None, None, 1, None, 1, 1, 1, None, None) == -1
    assert lib.plh_fp8_quantize(None, None, 0, 1, 1, 1, 1, None, None) == -1
    assert lib.plh_fp8_linear(None, None, 0, 1, 1, 1, None, 1e-5, None, None, 1, None, 1, None, 0) == -1
    assert lib.plh_fp8_ws_bytes(None, 1, 1, 1) == -1
    assert lib.plh_fp8_codes_bytes(0, 1) == -1 and lib.plh_fp8_codes_bytes(1, 0) == -1
    assert lib.plh_fp8_codes_bytes(33, 129) == 64 * 256
    header = (_native.LIB_PATH.parents[1] / "include" / "pagellm_hip.h").read_text()
    for name in ("PLH_BF16", "PLH_F16", "PLH_MAX_TOP"):
        assert f"#define {name} {getattr(_native, name)}\n" in header


def test_token_logits_without_a_context():
    lib = _native.load_library()
    assert lib.plh_token_logits(None, None, 0, 1, 1, 1, None, None) == -1


def test_sizes_of_very_large_matrices():
    lib = _native.load_library()
    for V, D in [(2**31 - 1, 1), (1, 2**31 - 1), (2**31 - 31, 129), (2**31 - 1, 2**31 - 1), (2**28, 128)]:
        assert lib.plh_fp8_codes_bytes(V, D) == -(-V // 32) * -(-D // 128) * 4096, (V, D)


def test_stage_without_a_context():
    lib = _native.load_library()
    assert lib.plh_stage(None, None, 8) == -1
    assert lib.plh_stage_h2d(None, None, None, 0) == -1
