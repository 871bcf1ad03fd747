"""Batched sampling for the engine's step loop, with device-resident histories.

``LLMEngine.step`` (``src/pagellm/engine/llm_engine.py:238-254``) calls
``_append_token`` once per finished sequence, and each call samples one row
with the sequence's full token history (``sample(logits, params, seq.rng,
seq.tokens)``, ``:283``) and then appends the token (``:284``).  The
:class:`BatchSampler` here replaces those per-row calls with one launch per
step:

* the histories live in HBM (:class:`DeviceHistories`), one fixed slot per
  sequence, and grow in place by one id per step on the device
  (``plh_append_ids``, reading the ids the sampler just wrote) instead of
  being re-uploaded every step;
* each sequence keeps its own numpy ``Generator`` on the host: one
  ``rng.random()`` per non-greedy row, none for greedy rows, in row order,
  exactly as the per-row loop consumes them (``sampling.py:98``, ``:102-106``);
* only the token ids come back to the host, with their log probabilities where
  a step asks for them.

Forked sequences (``SamplingParams.n > 1``, ``llm_engine.py:259-278``) join
with the parent's token list at the time of the fork, so each child samples
against its own copy of the history, as in the reference.
"""

from __future__ import annotations

from typing import Hashable, Sequence

import numpy as np

from . import _native
from .logits import DeviceLogprobs, _check_mask, _expand_rules, _pack_rules
from .sampling import _draw_uniforms, _expand_params, _history_ids, _is_torch_cuda, _nucleus_hint, _pack_params

__all__ = ["BatchSampler", "DeviceHistories"]


class DeviceHistories:
    """Token histories (prompt + outputs) of live sequences in HBM.

    One slot of ``max_len`` int32 ids per sequence in a single device slab;
    row b of a step reads ``slab[slot * max_len : slot * max_len + length]``
    through the sampler's span form of the history (``PLH_SAMPLE_HIST_SPANS``).
    """

    def __init__(self, vocab_size: int, max_seqs: int, max_len: int, *, ctx: _native.Context | None = None):
        if max_seqs < 1 or max_len < 1:
            raise ValueError("max_seqs and max_len must be >= 1")
        self.ctx = ctx if ctx is not None else _native.default_context()
        self.V = int(vocab_size)
        self.max_seqs = int(max_seqs)
        self.max_len = int(max_len)
        self.slab = self.ctx.empty((self.max_seqs * self.max_len,), np.int32)
        self._free = list(range(self.max_seqs - 1, -1, -1))
        self._slot: dict[Hashable, int] = {}
        self._len: dict[Hashable, int] = {}
        self._prompt: dict[Hashable, int] = {}  # where each sequence's outputs begin

    def __contains__(self, key) -> bool:
        return key in self._slot

    def __len__(self) -> int:
        return len(self._slot)

    def length(self, key) -> int:
        return self._len[key]

    def add(self, key, tokens, prompt_len: int | None = None) -> None:
        """A new sequence (or a fork) with its current token list, the first
        ``prompt_len`` of which (None: all) are its prompt: frequency and
        presence penalties count the tokens after them."""
        if key in self._slot:
            raise ValueError(f"sequence {key!r} already has a history")
        ids = _history_ids(tokens, self.V)
        if ids.size > self.max_len:
            raise ValueError(f"history of {ids.size} tokens exceeds max_len {self.max_len}")
        if prompt_len is not None and not 0 <= prompt_len <= ids.size:
            raise ValueError(f"prompt_len must be in [0, {ids.size}]")
        if not self._free:
            raise RuntimeError(f"all {self.max_seqs} history slots are in use")
        slot = self._free.pop()
        if ids.size:
            c = self.ctx
            c._check(c.lib.plh_h2d(c.handle, self.slab.ptr + 4 * slot * self.max_len, ids.ctypes.data, ids.nbytes))
        self._slot[key] = slot
        self._len[key] = int(ids.size)
        self._prompt[key] = int(ids.size if prompt_len is None else prompt_len)

    def remove(self, key) -> None:
        """A finished or aborted sequence gives its slot back."""
        slot = self._slot.pop(key)
        del self._len[key]
        del self._prompt[key]
        self._free.append(slot)

    def download(self, key) -> np.ndarray:
        """The sequence's history as the device holds it (for checks)."""
        n = self._len[key]
        out = np.empty(n, dtype=np.int32)
        if n:
            c = self.ctx
            c._check(c.lib.plh_d2h(c.handle, out.ctypes.data, self.slab.ptr + 4 * self._slot[key] * self.max_len,
                                   out.nbytes))
        return out

    def _slots_lengths(self, keys: Sequence) -> tuple[np.ndarray, np.ndarray]:
        B = len(keys)
        slots = np.fromiter(map(self._slot.__getitem__, keys), dtype=np.int64, count=B)
        lens = np.fromiter(map(self._len.__getitem__, keys), dtype=np.int64, count=B)
        return slots, lens

    def spans(self, keys: Sequence, active: Sequence[bool]) -> np.ndarray:
        """int64 [2B] (start, end) per row; inactive rows get an empty span."""
        slots, lens = self._slots_lengths(keys)
        sp = np.empty(2 * len(keys), dtype=np.int64)
        sp[0::2] = slots * self.max_len
        sp[1::2] = sp[0::2] + np.where(np.asarray(active, dtype=bool), lens, 0)
        return sp

    def spans_and_positions(self, keys: Sequence, active) -> tuple[np.ndarray, np.ndarray]:
        """spans(keys, active) and append_positions(keys) in one pass."""
        slots, lens = self._slots_lengths(keys)
        full = lens >= self.max_len
        if full.any():
            key = keys[int(np.argmax(full))]
            raise RuntimeError(f"history of {key!r} is full ({self.max_len} tokens)")
        start = slots * self.max_len
        sp = np.empty(2 * len(keys), dtype=np.int64)
        sp[0::2] = start
        sp[1::2] = start + np.where(np.asarray(active, dtype=bool), lens, 0)
        return sp, start + lens

    def append_positions(self, keys: Sequence) -> np.ndarray:
        """int64 [B]: where each row's next id goes."""
        slots, lens = self._slots_lengths(keys)
        full = lens >= self.max_len
        if full.any():
            key = keys[int(np.argmax(full))]
            raise RuntimeError(f"history of {key!r} is full ({self.max_len} tokens)")
        return slots * self.max_len + lens

    def output_starts(self, keys: Sequence) -> np.ndarray:
        """int64 [B]: where in its history each row's outputs begin."""
        return np.fromiter(map(self._prompt.__getitem__, keys), dtype=np.int64, count=len(keys))

    def advance(self, keys: Sequence) -> None:
        for key in keys:
            self._len[key] += 1


class BatchSampler:
    """One sampler launch per engine step over the rows of finished
    sequences (``llm_engine.py:238-254``), histories kept in HBM."""

    def __init__(self, histories: DeviceHistories):
        self.hist = histories
        self.ctx = histories.ctx
        # the last step's packed parameters, with references to its
        # SamplingParams objects (so that equal ids mean the same objects)
        self._packed = None

    def sample(self, logits, params, rngs: Sequence | None, keys: Sequence, *, uniforms=None, rules=None, masks=None,
               mask_rows=None, logprobs: int | None = None):
        """Samples one token per row and appends it to the row's history.

        ``logits`` is [B, V] (numpy, or a torch CUDA tensor read in place on
        torch's current stream); ``params`` one SamplingParams or one per
        row; ``rngs[b]`` row b's Generator (None allowed for greedy rows);
        ``keys[b]`` the sequence of row b, which must be in the histories.
        Returns int64 ids [B].

        ``rules`` (one :class:`pagellm_amd.logits.LogitRules`, or one or None per
        row) and ``masks`` with ``mask_rows`` (as ``process_logits`` takes them)
        are applied to a copy of the logits first: biases, then the repetition
        penalty, then frequency and presence penalties over the row's outputs
        (``DeviceHistories.add``'s ``prompt_len``), then the mask.  Rows without
        rules keep the sampler's own repetition penalty, and so their ids,
        whatever rows stand beside them.  A row whose rules and mask leave no
        token (-inf everywhere) gives the id -1 and joins no history; its
        Generator has moved like any other row's.  With ``logprobs`` = n the call
        returns (ids, :class:`pagellm_amd.logits.Logprobs`): the sampled tokens'
        log probabilities and ranks (NaN and 0 for an id of -1) and the n best
        tokens under the logits as given.
        """
        c = self.ctx
        B = len(keys)
        n_top = 0 if logprobs is None else int(logprobs)
        if not 0 <= n_top <= min(self.hist.V, _native.PLH_MAX_TOP):
            raise ValueError(f"logprobs must be in [0, {min(self.hist.V, _native.PLH_MAX_TOP)}]")
        process = rules is not None or masks is not None or mask_rows is not None
        if process:
            # refused here, before a Generator moves
            masks, mask_rows = _check_mask(masks, mask_rows, B, self.hist.V, c.device, _is_torch_cuda(logits))
            rules = _expand_rules(rules, B)
            f, pr, bias_ids, bias, bias_off = _pack_rules(rules, self.hist.V)
            ruled = np.array([not rule.neutral for rule in rules], dtype=bool)
            process = masks is not None or bool(ruled.any())
            # the rows whose tokens may all be ruled out
            masked = masks is not None if mask_rows is None else mask_rows >= 0
            closed = ruled | masked
        if B == 0:
            ids = np.zeros(0, dtype=np.int64)
            return ids if logprobs is None else (ids, DeviceLogprobs(c, 0, n_top, np.float32).download())
        if _is_torch_cuda(logits):
            import torch

            if logits.dim() != 2 or logits.stride(1) != 1 or int(logits.shape[0]) != B:
                raise ValueError("logits must be [B, V] with unit stride in the vocabulary dimension")
            if logits.dtype not in (torch.float32, torch.float64):
                raise TypeError("torch logits must be float32 or float64")
            if (process or logprobs is not None) and logits.device.index != c.device:
                raise ValueError(f"logits are on GPU {logits.device.index}, the context on GPU {c.device}")
            V = int(logits.shape[1])
            ptr, ld = logits.data_ptr(), int(logits.stride(0))
            code = _native.PLH_F64 if logits.dtype == torch.float64 else _native.PLH_F32
            c.set_stream(torch.cuda.current_stream(logits.device).cuda_stream)
        else:
            host = np.asarray(logits)
            if host.dtype != np.float32 and host.dtype != np.float64:
                host = host.astype(np.float64)
            host = np.ascontiguousarray(host)
            if host.ndim != 2 or host.shape[0] != B:
                raise ValueError("logits must be [B, V]")
            V = host.shape[1]
            dev, ld = c.upload_rows("eng_logits", host)
            ptr, code = dev.ptr, _native.dtype_code(host.dtype)
            c.set_stream(None)
        if V != self.hist.V:
            raise ValueError(f"vocabulary {V} does not match the histories' {self.hist.V}")
        params = _expand_params(params, B)
        u = (np.asarray(uniforms, dtype=np.float64).reshape(B) if uniforms is not None
             else _draw_uniforms(params, rngs, B))
        ids = list(map(id, params))
        if self._packed is not None and self._packed[0] == ids:
            t, k, p, r = self._packed[2]  # the same requests in the same rows as the last step
        else:
            t, k, p, r = _pack_params(params)
            self._packed = (ids, list(params), (t, k, p, r))
        # sampling.py:56: only rows whose penalty is active read their history
        # (for rows with rules the processing applies it, ahead of the sampler)
        own_r = np.where(ruled, 1.0, r) if process else r
        spans, pos = self.hist.spans_and_positions(keys, own_r != 1.0)
        # every per-row array in one page-locked host buffer, one queued copy
        # to the device (the download of the ids below waits for it)
        parts = [t, p, own_r, u, spans, pos, k]
        if process:
            rule_spans = self.hist.spans(keys, ruled & ((r != 1.0) | (f != 0.0) | (pr != 0.0)))
            host = [np.where(ruled, r, 1.0), f, pr, rule_spans, self.hist.output_starts(keys), bias, bias_off,
                    bias_ids, mask_rows, masks if isinstance(masks, np.ndarray) else None]
            parts += [a for a in host if a is not None]
        offs = np.cumsum([0] + [(a.nbytes + 7) & ~7 for a in parts])
        stage = c.pinned("eng_stage", int(offs[-1]))
        for a, o in zip(parts, offs[:-1]):
            stage[o:o + a.nbytes] = np.ascontiguousarray(a).reshape(-1).view(np.uint8)
        d = c.scratch("eng_stage", (int(offs[-1]),), np.uint8)
        c.h2d_async(d.ptr, stage[:int(offs[-1])])
        d_t, d_p, d_r, d_u, d_sp, d_pos, d_k = (d.ptr + int(o) for o in offs[:7])
        given, given_ld = ptr, ld
        if process:
            rest = iter(d.ptr + int(o) for o in offs[7:-1])
            h_r, h_f, h_p, h_sp, h_st, h_b, h_bo, h_bi, h_mr, h_m = (next(rest) if a is not None else None for a in host)
            mask_ld = n_masks = 0
            if masks is not None:
                n_masks, mask_ld = int(masks.shape[0]), int(masks.shape[1])
                if not isinstance(masks, np.ndarray):
                    h_m, mask_ld = masks.data_ptr(), int(masks.stride(0)) if n_masks > 1 else mask_ld
                if n_masks == 0:
                    h_m = None
            es = 8 if code == _native.PLH_F64 else 4
            ld = -(-V * es // 16) * 16 // es
            work = c.scratch("eng_processed", (B, ld), np.float64 if es == 8 else np.float32)
            ptr = work.ptr
            c.process_logits(given, code, given_ld, B, V, self.hist.slab.ptr, h_sp, h_st, h_r, h_f, h_p, h_bi, h_b,
                             h_bo, h_m, mask_ld, n_masks, h_mr, ptr, ld, _native.PLH_SAMPLE_HIST_SPANS)
        # the ids and, with rules, behind them their processed logits
        at = (4 * B + 7) & ~7
        value = np.dtype(np.float64 if code == _native.PLH_F64 else np.float32)
        out = c.scratch("eng_out", (at + value.itemsize * B if process else 4 * B,), np.uint8)
        c.sample(ptr, code, ld, B, V, self.hist.slab.ptr, d_sp, d_t, d_k, d_p, d_r, d_u,
                 out.ptr, None, _native.PLH_SAMPLE_HIST_SPANS | _nucleus_hint(t, k, p, V))
        # llm_engine.py:284: the token joins the history, on the device
        c.append_ids(self.hist.slab.ptr, d_pos, out.ptr, B)
        if process:
            c.token_logits(ptr, code, ld, B, V, out.ptr, out.ptr + at)
        if logprobs is not None:
            res = DeviceLogprobs(c, B, n_top, value)
            c.logprobs(given, code, given_ld, B, V, out.ptr, *res.pointers())
        raw = out.download()
        ids = raw[:4 * B].view(np.int32).astype(np.int64)
        lps = res.download() if logprobs is not None else None
        if process:
            # the sampler takes a token at -inf only where there is no other
            none = closed & np.isneginf(raw[at:].view(value))
            if none.any():
                ids[none] = -1
                if lps is not None:
                    lps.logprob[none] = np.nan
                    lps.rank[none] = 0
                keys = [key for key, left in zip(keys, ~none) if left]
        self.hist.advance(keys)
        return ids if logprobs is None else (ids, lps)
