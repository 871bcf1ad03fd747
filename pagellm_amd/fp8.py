"""The logits producer with 8-bit weights: e4m3 codes and a scale for each block.

:class:`pagellm_amd.head.LogitsHead` keeps lm_head in float32, and a decode step
of a few rows is bound by reading it once.  :class:`Fp8LogitsHead` keeps it in
OCP e4m3 with one float32 scale for each 128 x 128 block, a quarter of the
bytes, and rounds the rows of a call to e4m3 with a scale for each 128 of a row:

    head = Fp8LogitsHead(w["norm"], w["lm_head"], cfg.norm_eps)             # rounded once
    head = Fp8LogitsHead.from_codes(norm, codes, scales, cfg.norm_eps)      # an e4m3 checkpoint
    ids = sampler.sample(head(h), params, rngs, keys)                       # no host copy

It replaces ``rms_norm(h, self.w["norm"], eps) @ self.w["lm_head"]``
(``src/pagellm/model/transformer.py:271``) where the weights' rounding (at most
2^-4 of a value) is wanted; the reference has no 8-bit weights.  Tensors are
torch CUDA tensors on the context's GPU, read and written in place on torch's
current stream; weights may also come as numpy arrays.
"""

from __future__ import annotations

import numpy as np

from . import _native
from .sampling import _is_torch_cuda, _stream_of

__all__ = ["Fp8LogitsHead", "Fp8Weights", "fp8_linear"]

BLOCK = 128


def _ctx(ctx):
    return ctx if ctx is not None else _native.default_context()


def _float_code(x, name: str) -> int:
    import torch

    code = {torch.float32: _native.PLH_F32, torch.bfloat16: _native.PLH_BF16, torch.float16: _native.PLH_F16}.get(x.dtype)
    if code is None:
        raise TypeError(f"{name} must be float32, bfloat16 or float16")
    return code


def _check_device(c, x, name: str) -> None:
    if not _is_torch_cuda(x):
        raise TypeError(f"{name} must be a torch CUDA tensor")
    if x.device.index != c.device:
        raise ValueError(f"{name} is on GPU {x.device.index}, the context on GPU {c.device}")


def _on_device(x, c, dtype=None):
    """x as a tensor on the context's GPU (numpy arrays and CPU tensors are uploaded)."""
    import torch

    if not isinstance(x, torch.Tensor):
        x = torch.from_numpy(np.ascontiguousarray(x))
    return x.to(device=torch.device("cuda", c.device), dtype=dtype)


class Fp8Weights:
    """A [V, D] matrix in e4m3, laid out for the product kernels.

    ``codes`` (uint8) holds tiles of 32 rows x 128 columns, each in the order in
    which a wave reads it; ``scales`` is float32 [ceil(V / 128), ceil(D / 128)].
    """

    def __init__(self, V: int, D: int, ctx: _native.Context):
        import torch

        self.ctx, self.V, self.D = ctx, int(V), int(D)
        if self.V < 1 or self.D < 1:
            raise ValueError("the matrix must be [V, D] with V, D >= 1")
        if max(self.V, self.D) > 2**31 - 1:  # ctypes would wrap them
            raise ValueError("at most 2^31 - 1 rows and columns")
        dev = torch.device("cuda", ctx.device)
        nbytes = int(ctx.lib.plh_fp8_codes_bytes(self.V, self.D))
        self.codes = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        self.scales = torch.empty((-(-self.V // BLOCK), -(-self.D // BLOCK)), dtype=torch.float32, device=dev)

    @classmethod
    def quantize(cls, matrix, *, ctx: _native.Context | None = None) -> "Fp8Weights":
        """Rounds ``matrix`` [V, D] (float32, bfloat16 or float16, any strides):
        a block's scale is the smallest power of two s with max|w| <= 448 s, its
        codes the e4m3 values nearest to w / s, ties to even."""
        import torch

        c = _ctx(ctx)
        w = _on_device(matrix, c)
        if w.dim() != 2:
            raise ValueError("the matrix must be [V, D]")
        if w.dtype == torch.float64:
            raise TypeError("the matrix must be float32, bfloat16 or float16")
        code = _float_code(w, "the matrix")
        out = cls(w.shape[0], w.shape[1], c)
        c.set_stream(_stream_of(w))
        c.fp8_quantize(w.data_ptr(), code, int(w.stride(0)), int(w.stride(1)), out.V, out.D, out.codes.data_ptr(),
                       out.scales.data_ptr())
        return out

    @classmethod
    def from_codes(cls, codes, scales, *, ctx: _native.Context | None = None) -> "Fp8Weights":
        """Lays out a checkpoint's ``codes`` [V, D] (float8_e4m3fn, or their
        bytes as uint8) and ``scales`` [ceil(V / 128), ceil(D / 128)] float32."""
        import torch

        c = _ctx(ctx)
        q, s = _on_device(codes, c), _on_device(scales, c)
        if q.dtype not in (torch.float8_e4m3fn, torch.uint8):
            raise TypeError("codes must be float8_e4m3fn or uint8")
        if s.dtype != torch.float32:
            raise TypeError("scales must be float32")
        if q.dim() != 2:
            raise ValueError("codes must be [V, D]")
        out = cls(q.shape[0], q.shape[1], c)
        if tuple(s.shape) != tuple(out.scales.shape):
            raise ValueError(f"scales must be {list(out.scales.shape)} for codes {list(q.shape)}, got {list(s.shape)}")
        q = q if q.stride(1) == 1 and q.stride(0) >= out.D else q.contiguous()
        s = s.contiguous()
        c.set_stream(_stream_of(q))
        c.fp8_pack(q.data_ptr(), max(int(q.stride(0)), out.D), s.data_ptr(), int(s.shape[1]), out.V, out.D,
                   out.codes.data_ptr(), out.scales.data_ptr())
        return out

    def dequantize(self):
        """The matrix the codes stand for, float32 [V, D] on the GPU."""
        import torch

        vt, kb = -(-self.V // 32), -(-self.D // BLOCK)
        # a tile's order: 16 codes of k = 16 p .. of each of its rows, p = 0 .. 7
        q = self.codes.view(vt, kb, 8, 32, 16).permute(0, 3, 1, 2, 4).reshape(vt * 32, kb * BLOCK)
        w = q.contiguous().view(torch.float8_e4m3fn)[: self.V, : self.D].float()
        s = self.scales.repeat_interleave(BLOCK, 0)[: self.V].repeat_interleave(BLOCK, 1)[:, : self.D]
        return w * s


def fp8_linear(x, weights: Fp8Weights, *, norm=None, eps: float = 1e-5, out=None, ctx: _native.Context | None = None):
    """``y @ w.T`` in float32 with y the rows x [N, D] (after ``rms_norm(x, norm,
    eps)`` where ``norm`` is given) rounded to e4m3 in blocks of 128 of a row,
    and w the weights: [N, V] float32, in ``out`` (a new tensor when None; a
    row-strided view of a larger buffer is fine).  x is float32, bfloat16 or
    float16 with unit stride in its last dimension."""
    import torch

    c = ctx if ctx is not None else weights.ctx
    _check_device(c, x, "x")
    _check_device(c, weights.codes, "weights")
    code = _float_code(x, "x")
    if x.dim() != 2 or int(x.shape[1]) != weights.D:
        raise ValueError(f"x must be [N, {weights.D}]")
    N, V = int(x.shape[0]), weights.V
    if N > 2**31 - 1:  # ctypes would wrap it
        raise ValueError("at most 2^31 - 1 rows")
    if x.numel() and x.stride(1) != 1 and weights.D > 1:
        raise ValueError("x must have unit stride in its last dimension")
    if norm is not None:
        _check_device(c, norm, "norm")
        if norm.dtype != torch.float32:
            raise TypeError("norm must be float32")
        if tuple(norm.shape) != (weights.D,) or (weights.D > 1 and norm.stride(0) != 1):
            raise ValueError(f"norm must be [{weights.D}] with unit stride")
    if out is None:
        out = torch.empty((N, V), dtype=torch.float32, device=x.device)
    else:
        _check_device(c, out, "out")
        if out.dtype != torch.float32:
            raise TypeError("out must be float32")
        if tuple(out.shape) != (N, V) or (out.numel() and V > 1 and out.stride(1) != 1):
            raise ValueError(f"out must be [{N}, {V}] with unit stride in its last dimension")
        if N > 1 and out.stride(0) < V:
            raise ValueError("rows of out must not overlap")
    if N == 0:
        return out
    c.set_stream(_stream_of(x))
    nbytes = c.fp8_ws_bytes(N, V, weights.D)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)  # torch's allocator orders its reuse on the stream
    ldx = int(x.stride(0)) if N > 1 else weights.D
    ldo = int(out.stride(0)) if N > 1 else V
    c.fp8_linear(x.data_ptr(), code, ldx, N, weights.D, norm.data_ptr() if norm is not None else None, float(eps),
                 weights.codes.data_ptr(), weights.scales.data_ptr(), V, out.data_ptr(), ldo, ws.data_ptr(), nbytes)
    return out


class Fp8LogitsHead:
    """:class:`pagellm_amd.head.LogitsHead` with its lm_head in e4m3: calling it
    with the last hidden states of a step (float32, bfloat16 or float16) returns
    that step's float32 logits on the device."""

    def __init__(self, norm, lm_head, eps: float = 1e-5, *, ctx: _native.Context | None = None):
        """``lm_head`` is the reference's [D, V] (``transformer.py:184-197``)."""
        c = _ctx(ctx)
        if isinstance(lm_head, np.ndarray) and lm_head.dtype == np.float64:
            lm_head = lm_head.astype(np.float32)  # as LogitsHead takes it
        w = _on_device(lm_head, c)
        if w.dim() != 2:
            raise ValueError("lm_head must be [D, V]")
        self._init(norm, Fp8Weights.quantize(w.T, ctx=c), eps)

    def _init(self, norm, weights: Fp8Weights, eps: float) -> None:
        import torch

        self.ctx, self.weights, self.eps = weights.ctx, weights, float(eps)
        self.D, self.V = weights.D, weights.V
        self.norm = _on_device(norm, self.ctx, torch.float32).contiguous()
        if tuple(self.norm.shape) != (self.D,):
            raise ValueError(f"norm must be [{self.D}]")

    @classmethod
    def from_codes(cls, norm, codes, scales, eps: float = 1e-5, *, ctx: _native.Context | None = None) -> "Fp8LogitsHead":
        """From a checkpoint's e4m3 ``codes`` [V, D] and float32 ``scales`` of
        their 128 x 128 blocks (:meth:`Fp8Weights.from_codes`)."""
        head = cls.__new__(cls)
        head._init(norm, Fp8Weights.from_codes(codes, scales, ctx=ctx), eps)
        return head

    def __call__(self, h, out=None):
        if not _is_torch_cuda(h):
            h = _on_device(np.ascontiguousarray(h, dtype=np.float32), self.ctx)
        return fp8_linear(h, self.weights, norm=self.norm, eps=self.eps, out=out)
