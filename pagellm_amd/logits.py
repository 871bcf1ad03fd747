"""What a request asks of its logits beside sampling, computed on MI355X.

* :func:`process_logits`: biases, repetition, frequency and presence penalties
  and grammar masks on a batch's logits (``plh_process_logits``).  The reference
  has the repetition penalty alone (``src/pagellm/engine/sampling.py:52-62``).
* :func:`token_logprobs`: each row's log probability and rank of its chosen
  token, and its best tokens with theirs (``plh_logprobs``).

Logits may be numpy arrays (uploaded, and the results downloaded) or torch CUDA
tensors (read and written in place on torch's current stream; results stay on
the GPU and the host waits for nothing: rules, masks and ids that are on the host
go over in a queued copy, which a graph cannot capture).
:class:`pagellm_amd.engine.BatchSampler` takes the same rules and masks and returns
the same log probabilities for an engine's step.
"""

from __future__ import annotations

import math
from dataclasses import dataclass, field
from typing import Iterable, Mapping, NamedTuple, Sequence

import numpy as np

from . import _native
from .sampling import _as_float_rows, _ctx, _expand_params, _history_ids, _int64_row, _is_torch_cuda, _stream_of

__all__ = ["LogitRules", "Logprobs", "pack_mask", "process_logits", "token_logprobs"]


@dataclass(frozen=True)
class LogitRules:
    """One request's rules beside its ``SamplingParams``.

    ``frequency_penalty`` is taken off a token's logit once for each time it
    occurs among the request's outputs, ``presence_penalty`` once if it occurs
    at all; ``logit_bias`` maps token ids to what is added to their logits
    (-inf rules a token out).  The mapping is packed here: changing it later
    changes nothing."""

    frequency_penalty: float = 0.0
    presence_penalty: float = 0.0
    logit_bias: Mapping[int, float] = field(default_factory=dict, hash=False)

    def __post_init__(self) -> None:
        if not math.isfinite(self.frequency_penalty):
            raise ValueError("frequency_penalty must be finite")
        if not math.isfinite(self.presence_penalty):
            raise ValueError("presence_penalty must be finite")
        bias = {int(t): float(v) for t, v in dict(self.logit_bias).items()}
        if any(t < 0 or t > 2**31 - 1 for t in bias):
            raise ValueError("logit_bias needs token ids >= 0")
        if any(math.isnan(v) or v == math.inf for v in bias.values()):
            raise ValueError("logit_bias must be finite or -inf")
        object.__setattr__(self, "logit_bias", bias)
        # packed once: a batch's list is a concatenation
        object.__setattr__(self, "_ids", np.fromiter(bias.keys(), dtype=np.int32, count=len(bias)))
        object.__setattr__(self, "_values", np.fromiter(bias.values(), dtype=np.float64, count=len(bias)))
        object.__setattr__(self, "_last", max(bias, default=-1))

    @property
    def penalises(self) -> bool:
        return self.frequency_penalty != 0.0 or self.presence_penalty != 0.0

    @property
    def neutral(self) -> bool:
        return not self.penalises and not self.logit_bias


_NO_RULES = LogitRules()


class Logprobs(NamedTuple):
    """``logprob`` [B] and ``rank`` [B] (1: the best) of the chosen tokens (None
    without them), ``top_ids`` and ``top_logprobs`` [B, n] of the best."""

    logprob: object
    rank: object
    top_ids: object
    top_logprobs: object


def mask_words(V: int) -> int:
    """32-bit words of one mask row."""
    return (V + 31) // 32


def pack_mask(allowed, V: int) -> np.ndarray:
    """uint32 [ceil(V / 32)]: one row of a mask from the allowed token ids, or
    from a boolean array of V entries."""
    bits = np.zeros(mask_words(V) * 32, dtype=np.uint8)
    a = np.asarray(allowed if isinstance(allowed, np.ndarray) else list(allowed))
    if a.dtype == np.bool_:
        if a.shape != (V,):
            raise ValueError(f"expected {V} truth values")
        bits[:V] = a
    elif a.size:
        bits[_history_ids(a, V)] = 1
    return np.packbits(bits, bitorder="little").view("<u4")


def _expand_rules(rules, B: int) -> list[LogitRules]:
    if rules is None:
        return [_NO_RULES] * B
    if isinstance(rules, LogitRules):
        return [rules] * B
    rules = [r if r is not None else _NO_RULES for r in rules]
    if len(rules) != B:
        raise ValueError(f"expected {B} LogitRules, got {len(rules)}")
    return rules


def _pack_rules(rules: Sequence[LogitRules], V: int):
    """(frequency, presence, bias ids, biases, bias offsets) of a batch; the
    last three None without biases."""
    f = np.array([r.frequency_penalty for r in rules], dtype=np.float64)
    p = np.array([r.presence_penalty for r in rules], dtype=np.float64)
    if all(r._last < 0 for r in rules):
        return f, p, None, None, None
    for r in rules:
        if r._last >= V:
            raise IndexError(f"logit_bias of token {r._last} is out of bounds for a vocabulary of {V}")
    off = np.cumsum([0] + [r._ids.size for r in rules], dtype=np.int64)
    return f, p, np.concatenate([r._ids for r in rules]), np.concatenate([r._values for r in rules]), off


def _check_sizes(B: int, V: int) -> None:
    if V == 0:
        raise ValueError("empty vocabulary")
    if max(B, V) > 2**31 - 1:  # ctypes would wrap them
        raise ValueError("at most 2^31 - 1 rows and tokens")


def _check_mask(masks, mask_rows, B: int, V: int, device: int, logits_on_gpu: bool):
    """(masks, per-row int32 mask rows or None) of a call; masks as a CUDA
    tensor or a contiguous uint32 array."""
    if masks is None:
        if mask_rows is not None:
            raise ValueError("mask_rows given without masks")
        return None, None
    if _is_torch_cuda(masks):
        import torch

        if not logits_on_gpu:  # these are processed on the context's stream, not on torch's
            raise TypeError("CUDA masks need CUDA logits")
        if masks.dtype not in (torch.int32, getattr(torch, "uint32", torch.int32)):
            raise TypeError("masks must be int32 or uint32 words")
        if masks.device.index != device:
            raise ValueError(f"masks are on GPU {masks.device.index}, the context on GPU {device}")
        if masks.dim() != 2 or masks.stride(1) != 1 and masks.shape[1] > 1:
            raise ValueError("masks must be [rows, words] with unit stride")
        if masks.shape[0] > 1 and masks.stride(0) < mask_words(V):
            raise ValueError("rows of masks must not overlap (let rows share one by mask_rows)")
    else:
        masks = np.asarray(masks)
        if masks.dtype not in (np.dtype(np.uint32), np.dtype(np.int32)):
            raise TypeError("masks must be int32 or uint32 words")
        if masks.ndim != 2:
            raise ValueError("masks must be [rows, words]")
        masks = np.ascontiguousarray(masks)
    if masks.shape[1] < mask_words(V):
        raise ValueError(f"masks need {mask_words(V)} words for a vocabulary of {V}")
    if mask_rows is None:
        if masks.shape[0] != B:
            raise ValueError(f"expected {B} mask rows, got {masks.shape[0]} (or give mask_rows)")
        return masks, None
    rows = np.array([-1 if m is None else int(m) for m in mask_rows], dtype=np.int64)
    if rows.size != B:
        raise ValueError(f"expected {B} mask_rows, got {rows.size}")
    if rows.size and (rows.max() >= masks.shape[0] or rows.min() < -1):
        raise IndexError(f"mask_rows must be None, -1 or in [0, {masks.shape[0]})")
    return masks, rows.astype(np.int32)


def _pack(parts, empty=lambda n: np.empty(n, dtype=np.uint8)) -> tuple[np.ndarray, list[int | None]]:
    """The host arrays in parts (None allowed) in one buffer, each 16-byte
    aligned, and their offsets; the buffer is empty(its bytes)."""
    arrs = [None if a is None else np.ascontiguousarray(a) for a in parts]
    offs, n = [], 0
    for a in arrs:
        offs.append(None if a is None else n)
        n += 0 if a is None else (a.nbytes + 15) & ~15
    buf = empty(max(n, 16))
    for a, o in zip(arrs, offs):
        if a is not None:
            buf[o:o + a.nbytes] = a.reshape(-1).view(np.uint8)
    return buf, offs


def process_logits(
    logits,
    rules=None,
    params=None,
    contexts: Sequence | None = None,
    *,
    prompt_lens: Iterable[int] | None = None,
    masks=None,
    mask_rows=None,
    out=None,
    ctx: _native.Context | None = None,
):
    """Applies, to each row of ``logits`` [B, V] in this order, the biases of its
    :class:`LogitRules`, the repetition penalty of its ``SamplingParams`` over its
    context, its frequency and presence penalties, and its mask.

    ``rules`` and ``params`` are one for all rows, one per row, or None;
    ``contexts[b]`` is row b's tokens (prompt + outputs), of which the first
    ``prompt_lens[b]`` are no outputs (None: all are outputs).  ``masks`` is
    uint32 (or int32) [M, >= ceil(V / 32)], bit v % 32 of word v / 32 set where
    token v is allowed; ``mask_rows[b]`` names row b's (None or -1: no mask), and
    without ``mask_rows`` row b's is row b.  Returns the processed logits: a new
    numpy array, or for a torch CUDA tensor ``out`` (a new tensor when None;
    ``logits`` itself changes it in place)."""
    c = _ctx(ctx)
    on_gpu = _is_torch_cuda(logits)
    if on_gpu:
        import torch

        if logits.dim() != 2 or (logits.numel() and logits.shape[1] > 1 and logits.stride(1) != 1):
            raise ValueError("logits must be a 2-D tensor with unit stride in the vocabulary dimension")
        if logits.dtype not in (torch.float32, torch.float64):
            raise TypeError("torch logits must be float32 or float64")
        if logits.device.index != c.device:
            raise ValueError(f"logits are on GPU {logits.device.index}, the context on GPU {c.device}")
        if out is None:
            out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        elif not _is_torch_cuda(out) or out.dtype != logits.dtype or out.shape != logits.shape or \
                out.device != logits.device or (out.numel() and out.shape[1] > 1 and out.stride(1) != 1):
            raise ValueError("out must be like logits, with unit stride in the vocabulary dimension")
    else:
        if out is not None:
            raise ValueError("out needs torch CUDA logits")
        logits = _as_float_rows(logits)
        if logits.ndim != 2:
            raise ValueError("logits must be [B, V]")
    B, V = int(logits.shape[0]), int(logits.shape[1])
    _check_sizes(B, V)
    rules = _expand_rules(rules, B)
    params = _expand_params(params, B) if params is not None else None
    masks, mask_rows = _check_mask(masks, mask_rows, B, V, c.device, on_gpu)
    f, p, bias_ids, bias, bias_off = _pack_rules(rules, V)
    r = np.array([sp.repetition_penalty for sp in params], dtype=np.float64) if params is not None else None
    hist_ids = hist_off = start = None
    if contexts is not None:
        if len(contexts) != B:
            raise ValueError(f"expected {B} contexts, got {len(contexts)}")
        reads = [rules[b].penalises or (r is not None and r[b] != 1.0) for b in range(B)]
        parts = [_history_ids(_int64_row(contexts[b]), V) if reads[b] and contexts[b] is not None
                 else np.zeros(0, np.int32) for b in range(B)]
        if prompt_lens is not None:
            start = np.array([int(n) for n in prompt_lens], dtype=np.int64)
            if start.size != B:
                raise ValueError(f"expected {B} prompt_lens, got {start.size}")
            if start.size and start.min() < 0:
                raise ValueError("prompt_lens must be >= 0")
        hist_off = np.cumsum([0] + [a.size for a in parts], dtype=np.int64)
        hist_ids = np.concatenate(parts) if parts else None
        if hist_off[-1] == 0:
            hist_ids = hist_off = start = None
    elif prompt_lens is not None:
        raise ValueError("prompt_lens given without contexts")
    if B == 0:
        return out if on_gpu else logits
    host_masks = masks if masks is not None and not _is_torch_cuda(masks) else None
    f, p = (a if a.any() else None for a in (f, p))
    r = r if r is not None and (r != 1.0).any() else None
    parts = [r, f, p, bias, bias_off, hist_off, start, bias_ids, hist_ids, mask_rows, host_masks]
    code = _native.PLH_F64 if "float64" in str(logits.dtype) else _native.PLH_F32
    if on_gpu:
        c.set_stream(_stream_of(logits))
        base, offs = 0, [None] * len(parts)
        if any(a is not None for a in parts):
            keep = None

            def empty(n):
                nonlocal keep  # first: what fails here leaves no staged memory given
                keep = torch.empty(n, dtype=torch.uint8, device=logits.device)
                return c.stage(n)

            buf, offs = _pack(parts, empty)
            base = keep.data_ptr()  # torch's allocator orders its reuse on the stream
            c.stage_h2d(base, buf)
        x, ld = logits.data_ptr(), int(logits.stride(0)) if B > 1 else V
        o, ldo = out.data_ptr(), int(out.stride(0)) if B > 1 else V
    else:
        buf, offs = _pack(parts)
        c.set_stream(None)
        base = c.scratch_upload("process_in", buf).ptr
        dev, ld = c.upload_rows("process_x", logits)
        x = o = dev.ptr
        ldo = ld
    d_r, d_f, d_p, d_b, d_bo, d_ho, d_st, d_bi, d_hi, d_mr, d_m = (None if i is None else base + i for i in offs)
    mask_ld, n_masks = (0, 0)
    if masks is not None:
        n_masks = int(masks.shape[0])
        mask_ld = int(masks.shape[1])
        if host_masks is None:
            d_m, mask_ld = masks.data_ptr(), int(masks.stride(0)) if n_masks > 1 else mask_ld
        if n_masks == 0:
            d_m = None  # no row of a batch names one
    c.process_logits(x, code, ld, B, V, d_hi, d_ho, d_st, d_r, d_f, d_p, d_bi, d_b, d_bo, d_m, mask_ld, n_masks, d_mr,
                     o, ldo)
    if on_gpu:
        return out
    dev.shape, dev.dtype = (B, ld), logits.dtype
    return np.ascontiguousarray(dev.download()[:, :V])


def token_logprobs(logits, ids=None, n_top: int = 0, *, ctx: _native.Context | None = None) -> Logprobs:
    """:class:`Logprobs` of ``logits`` [B, V]: x - logsumexp(x) of the tokens
    ``ids`` [B] and their ranks, and the ``n_top`` (at most 64) best tokens, by
    logit descending and then by id ascending, with theirs.  Results have the
    logits' type (ids and ranks int32): numpy for numpy logits, CUDA tensors,
    not waited for, for a CUDA tensor (whose ids then may be a CUDA tensor; an
    id outside the vocabulary gives NaN and rank 0)."""
    c = _ctx(ctx)
    on_gpu = _is_torch_cuda(logits)
    if on_gpu:
        import torch

        if logits.dim() != 2 or (logits.numel() and logits.shape[1] > 1 and logits.stride(1) != 1):
            raise ValueError("logits must be a 2-D tensor with unit stride in the vocabulary dimension")
        if logits.dtype not in (torch.float32, torch.float64):
            raise TypeError("torch logits must be float32 or float64")
        if logits.device.index != c.device:
            raise ValueError(f"logits are on GPU {logits.device.index}, the context on GPU {c.device}")
    else:
        logits = _as_float_rows(logits)
        if logits.ndim != 2:
            raise ValueError("logits must be [B, V]")
    B, V = int(logits.shape[0]), int(logits.shape[1])
    _check_sizes(B, V)
    n = int(n_top)
    if not 0 <= n <= min(V, _native.PLH_MAX_TOP):
        raise ValueError(f"n_top must be in [0, {min(V, _native.PLH_MAX_TOP)}]")
    if ids is not None and not _is_torch_cuda(ids):
        ids = np.asarray(ids, dtype=np.int64).reshape(-1)
        if ids.size and (ids.min() < 0 or ids.max() >= V):
            raise IndexError(f"ids must be in [0, {V})")
        ids = ids.astype(np.int32)
    if ids is not None and tuple(ids.shape) != (B,):
        raise ValueError(f"expected {B} ids")
    if on_gpu:
        c.set_stream(_stream_of(logits))
        if isinstance(ids, np.ndarray):
            host, ids = ids, torch.empty(B, dtype=torch.int32, device=logits.device)
            if B:
                buf = c.stage(host.nbytes)
                buf[:] = host.view(np.uint8)
                c.stage_h2d(ids.data_ptr(), buf)
        elif ids is not None:
            if ids.is_floating_point():
                raise TypeError("ids must be integers")
            # ids past int32 stay outside every vocabulary
            ids = ids.clamp(-1, 2**31 - 1) if ids.dtype == torch.int64 else ids
            ids = ids.to(device=logits.device, dtype=torch.int32).contiguous()
        new = lambda shape, dt: torch.empty(shape, dtype=dt, device=logits.device)  # noqa: E731
        res = Logprobs(new(B, logits.dtype) if ids is not None else None,
                       new(B, torch.int32) if ids is not None else None,
                       new((B, n), torch.int32), new((B, n), logits.dtype))
        if B == 0:
            return res
        code = _native.PLH_F64 if logits.dtype == torch.float64 else _native.PLH_F32
        ptr = lambda t: t.data_ptr() if t is not None and t.numel() else None  # noqa: E731
        c.logprobs(logits.data_ptr(), code, int(logits.stride(0)) if B > 1 else V, B, V, ptr(ids), ptr(res.logprob),
                   ptr(res.rank), n, ptr(res.top_ids), ptr(res.top_logprobs))
        return res
    dt = logits.dtype
    if B == 0:
        return Logprobs(np.empty(0, dt) if ids is not None else None, np.empty(0, np.int32) if ids is not None else None,
                        np.empty((0, n), np.int32), np.empty((0, n), dt))
    if _is_torch_cuda(ids):
        raise TypeError("CUDA ids need CUDA logits")
    c.set_stream(None)
    dev, ld = c.upload_rows("lp_x", logits)
    d_ids = c.scratch_upload("lp_ids", ids) if ids is not None else None
    res = DeviceLogprobs(c, B, n, dt)
    c.logprobs(dev.ptr, _native.dtype_code(dt), ld, B, V, d_ids.ptr if d_ids is not None else None, *res.pointers())
    got = res.download()
    return got if ids is not None else got._replace(logprob=None, rank=None)


class DeviceLogprobs:
    """The outputs of one ``plh_logprobs`` call in one reusable device buffer,
    downloaded together."""

    def __init__(self, c: _native.Context, B: int, n: int, dtype):
        self.B, self.n, self.dtype = B, n, np.dtype(dtype)
        e = self.dtype.itemsize
        # the wider type first, so that every part is aligned to its element
        self.offs = np.cumsum([0, e * B, e * B * n, 4 * B])
        self.buf = c.scratch("lp_out", (int(self.offs[-1]) + 4 * B * n,), np.uint8)

    def pointers(self):
        """(out_lp, out_rank, n_top, top_ids, top_lp) for ``Context.logprobs``."""
        lp, top_lp, rank, top_ids = (self.buf.ptr + int(o) for o in self.offs)
        return lp, rank, self.n, top_ids if self.n else None, top_lp if self.n else None

    def download(self) -> Logprobs:
        raw = self.buf.download()
        o, B, n = self.offs, self.B, self.n
        return Logprobs(raw[: o[1]].view(self.dtype), raw[o[2]:o[3]].view(np.int32),
                        raw[o[3]:].view(np.int32).reshape(B, n), raw[o[1]:o[2]].view(self.dtype).reshape(B, n))
