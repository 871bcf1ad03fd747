"""Products with e4m3 weights (``plh_fp8_*``) against the float64 oracle (needs
an MI355X).

Tolerance of a product: products of codes are exact, a block's 128 of them are
added in float32 in some order (at most 127 roundings of 2^-24 of the block's
magnitude, one more for its scale), then the blocks (one each): (128 + blocks) *
2^-24 of sum |a| |w|.  Codes are exact: rows against an identity come back as the
values that their codes stand for."""

from __future__ import annotations

import numpy as np
import pytest

import oracle
from oracle import fp8 as O
from pagellm_amd import _native
from pagellm_amd.fp8 import Fp8LogitsHead, Fp8Weights, fp8_linear

pytestmark = pytest.mark.gpu


def _tol(D):
    return (128 + -(-D // 128)) * 2.0 ** -24


def _matrix(g, V, D):
    """Weights whose size differs from block to block."""
    w = 0.02 * g.standard_normal((V, D))
    for v in range(0, V, 128):
        for d in range(0, D, 128):
            w[v:v + 128, d:d + 128] *= 2.0 ** g.normal(0, 1.5)
    return w.astype(np.float32)


def _cuda(x, dtype=None):
    import torch

    return torch.from_numpy(np.ascontiguousarray(x)).to(device="cuda", dtype=dtype)


def _check(got, ref, bound, D):
    got = got.double().cpu().numpy() if hasattr(got, "cpu") else got
    assert got.shape == ref.shape
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    ok = ~np.isnan(ref)
    err = np.abs(got - ref)[ok]
    assert np.all(err <= _tol(D) * bound[ok] + 1e-37), float((err / (bound[ok] + 1e-37)).max())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("V,D", [(1, 1), (16, 128), (17, 129), (128, 200), (300, 127), (130, 1000)])
def test_codes_of_a_matrix(V, D, dtype):
    """quantize of both layouts, against the oracle, exactly."""
    import torch

    print(f"[fp8] codes {V}x{D} {dtype}", flush=True)
    g = np.random.default_rng(V + D)
    w = _matrix(g, V, D)
    w[0, 0] = 0.0
    if V > 16 and D > 128:
        w[:, 128:] = 0.0             # blocks of zeros
        w[3, 5], w[9, 7] = np.nan, np.inf
        w[16, :3] = [1e-9, -448.0, 2.0 ** -20]
    t = _cuda(w, getattr(torch, dtype))
    want = O.round_matrix(t.double().cpu().numpy())
    wide = torch.full((D, V + 3), float("nan"), dtype=t.dtype, device="cuda")
    wide[:, 1:V + 1] = t.T
    for m in (t, wide[:, 1:V + 1].T):
        q = Fp8Weights.quantize(m)
        assert np.array_equal(q.dequantize().double().cpu().numpy(), want, equal_nan=True)


def test_codes_of_extreme_values():
    """Blocks at the ends of float32's range; every code and every midpoint."""
    x = np.zeros((6, 256), dtype=np.float32)
    fin = np.sort(O.decode(np.arange(127)))
    x[0, :127], x[0, 128:254] = fin, (fin[1:] + fin[:-1]) / 2
    x[1] = -x[0]
    x[2] = np.float32(3e38) * np.linspace(-1, 1, 256, dtype=np.float32)
    x[3] = np.float32(2.0 ** -140) * np.arange(256)
    x[4, :128] = 448.0 * (1 + 2.0 ** -23)
    x[4, 128:] = 448.0
    x[5, 7] = 2.0 ** -149
    eye = Fp8Weights.from_codes(_cuda((np.eye(256) * 0x38).astype(np.uint8)),
                                _cuda(np.ones((2, 2), dtype=np.float32)))
    got = fp8_linear(_cuda(x), eye).double().cpu().numpy()
    want = O.round_rows(x)
    # a scaled value below float32's normal range may come back as zero or a subnormal
    small = np.abs(want) < 2.0 ** -126
    assert np.array_equal(got[~small], want[~small]) and np.all(np.abs(got[small]) <= 2.0 ** -126)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("N,D", [(1, 1), (5, 128), (16, 130), (33, 1000), (3, 8200)])
def test_codes_of_rows(N, D, dtype):
    """Rows with and without the norm, against the identity, exactly: the values
    that the oracle's codes stand for."""
    import torch

    print(f"[fp8] rows {N}x{D} {dtype}", flush=True)
    g = np.random.default_rng(N + D)
    x = _cuda(g.standard_normal((N, D)) * 2.0 ** g.normal(0, 2, (N, 1)), getattr(torch, dtype))
    norm = (1 + 0.1 * g.standard_normal(D)).astype(np.float32)
    take = np.unique(np.concatenate([[0, D - 1, D // 2], g.integers(0, D, 40)]))
    codes = np.zeros((take.size, D), dtype=np.uint8)
    codes[np.arange(take.size), take] = 0x38  # 1.0
    eye = Fp8Weights.from_codes(_cuda(codes), _cuda(np.ones((1, -(-D // 128)), dtype=np.float32)))
    host = x.double().cpu().numpy()
    got = fp8_linear(x, eye).double().cpu().numpy()
    assert np.array_equal(got, O.round_rows(host)[:, take])
    got = fp8_linear(x, eye, norm=_cuda(norm), eps=1e-5).double().cpu().numpy()
    assert np.array_equal(got, O.round_rows(O.norm_rows(host, norm, 1e-5))[:, take])


# rows: one, a tile, around tiles of 16, 64, 128 and 256, several of them
@pytest.mark.parametrize("N", [1, 2, 15, 16, 17, 32, 33, 64, 65, 127, 128, 129, 255, 256, 257, 300, 600])
@pytest.mark.parametrize("V,D", [
    (1, 1),
    (65, 128),       # the character vocabulary
    (127, 130),      # ragged everywhere
    (1000, 1000),
    (257, 4100),     # many blocks, the last ragged
    (4096, 256),
])
def test_product_matches_oracle(N, V, D):
    print(f"[fp8] product N={N} V={V} D={D}", flush=True)
    g = np.random.default_rng(N + 7 * V + D)
    x = g.standard_normal((N, D)).astype(np.float32)
    norm = (1 + 0.1 * g.standard_normal(D)).astype(np.float32)
    w = Fp8Weights.quantize(_cuda(_matrix(g, V, D)))
    ref, bound = O.linear(x, w.dequantize().double().cpu().numpy(), norm, 1e-5)
    _check(fp8_linear(_cuda(x), w, norm=_cuda(norm), eps=1e-5), ref, bound, D)


@pytest.mark.parametrize("N,V,D", [
    (300, 20011, 200),   # tiles of 128 rows, everything ragged
    (129, 50001, 130),
    (1100, 6007, 1537),  # more rows than run in ranges, k of 13 blocks
    (40, 2000, 1536),    # slices of k
    (200, 1000, 4000),
])
def test_tiles_and_slices(N, V, D):
    test_product_matches_oracle(N, V, D)


@pytest.mark.parametrize("N", [8, 40, 300])
@pytest.mark.parametrize("V,D", [(333, 200), (1024, 384)])
def test_strided_rows_and_outputs(N, V, D):
    """x and out as views of odd strides; nothing outside out is written; any
    float32 scales, negative and zero ones among them."""
    import torch

    print(f"[fp8] strides N={N} V={V} D={D}", flush=True)
    g = np.random.default_rng(N)
    codes = g.integers(0, 255, (V, D + 5)).astype(np.uint8)
    codes[(codes & 127) == 127] = 3
    scales = (g.standard_normal((-(-V // 128), -(-D // 128))) * 0.01).astype(np.float32)
    scales[0, 0] = 0.0
    w = Fp8Weights.from_codes(_cuda(codes)[:, :D], _cuda(scales))
    want = O.decode(codes[:, :D]) * np.repeat(np.repeat(scales.astype(np.float64), 128, 0)[:V], 128, 1)[:, :D]
    assert np.array_equal(w.dequantize().cpu().numpy(), want.astype(np.float32))
    xb = torch.full((N, D + 3), float("nan"), device="cuda", dtype=torch.bfloat16)
    xb[:, 1:D + 1] = torch.randn((N, D), device="cuda")
    ob = torch.full((N + 1, V + 5), 7.0, device="cuda")
    x = xb[:, 1:D + 1]
    fp8_linear(x, w, out=ob[:N, 1:V + 1])
    ref, bound = O.linear(x.double().cpu().numpy(), want)
    _check(ob[:N, 1:V + 1], ref, bound, D)
    assert bool((ob[N] == 7).all()) and bool((ob[:, 0] == 7).all()) and bool((ob[:, V + 1:] == 7).all())


@pytest.mark.parametrize("N", [3, 40, 300])
def test_nan_rows_and_columns_leave_the_others_alone(N):
    """A row with NaN or an infinity is NaN, a column with a NaN code too; every
    other output keeps its bits, and a row of zeros gives zeros."""
    import torch

    V, D = 400, 300
    g = np.random.default_rng(N)
    codes = g.integers(0, 127, (V, D)).astype(np.uint8)
    codes[codes == 127] = 0
    scales = np.full((4, 3), 0.01, dtype=np.float32)
    x = _cuda(g.standard_normal((N, D)).astype(np.float32))
    x[2] = 0.0
    ref = fp8_linear(x, Fp8Weights.from_codes(_cuda(codes), _cuda(scales)))
    assert bool((ref[2] == 0).all()) and bool(ref.isfinite().all())
    codes[17, 299] = 0xFF
    w = Fp8Weights.from_codes(_cuda(codes), _cuda(scales))
    for bad in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[1, 150] = bad
        for norm in (None, torch.ones(D, device="cuda")):
            got = fp8_linear(y, w, norm=norm)
            assert bool(got[1].isnan().all()) and bool(got[:, 17].isnan().all())
            if norm is None:
                keep = ref.clone()
                keep[1], keep[:, 17] = got[1], got[:, 17]
                assert torch.equal(got.nan_to_num(9), keep.nan_to_num(9))


def test_equal_calls_equal_bits_and_full_size():
    """256 x 4096 x 128 256 against torch's float32 product of the same codes."""
    import torch

    torch.manual_seed(0)
    N, D, V = 256, 4096, 128256
    print("[fp8] full size", flush=True)
    w = Fp8Weights.quantize(0.02 * torch.randn((V, D), device="cuda"))
    x = torch.randn((N, D), device="cuda", dtype=torch.bfloat16)
    eye = Fp8Weights.from_codes((torch.eye(D, device="cuda") * 0x38).to(torch.uint8),
                                torch.ones((32, 32), device="cuda"))
    a = fp8_linear(x, eye)
    got = fp8_linear(x, w)
    assert torch.equal(got, fp8_linear(x, w))
    full = w.dequantize()
    bound = a.abs() @ full.abs().T
    err = (got - a @ full.T).abs()
    # both sides round: twice the tolerance and 4096 roundings of the plain sum are far above what is seen
    worst = float((err / bound).max())
    print(f"[fp8] worst error / bound {worst:.3e}", flush=True)
    assert worst <= _tol(D) + D * 2.0 ** -24


def test_streams_and_graphs():
    """Two streams at once, and graphs replayed at once: each call has its own
    workspace."""
    import torch

    V, D = 3000, 1024
    g = np.random.default_rng(0)
    w = Fp8Weights.quantize(_cuda(_matrix(g, V, D)))
    xs = [torch.randn((n, D), device="cuda") for n in (8, 100)]
    want = [fp8_linear(x, w).clone() for x in xs]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, x in zip(streams, xs):
            with torch.cuda.stream(s):
                got.append(fp8_linear(x, w))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    outs = [torch.empty_like(o) for o in want]
    graphs = []
    for s, x, o in zip(streams, xs, outs):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=s):
            fp8_linear(x, w, out=o)
        graphs.append(gr)
    for i in range(3):
        for x in xs:
            x.normal_()
        torch.cuda.synchronize()
        for s, gr in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for x, o in zip(xs, outs):
            assert torch.equal(o, fp8_linear(x, w))


def test_head_and_refusals():
    import torch

    g = np.random.default_rng(5)
    D, V = 256, 1000
    norm = (1 + 0.1 * g.standard_normal(D)).astype(np.float32)
    lm_head = _matrix(g, V, D).T.copy()
    h = g.standard_normal((12, D)).astype(np.float32)
    head = Fp8LogitsHead(norm, lm_head, 1e-5)
    ref, bound = O.linear(h, O.round_matrix(lm_head.T), norm, 1e-5)
    _check(head(h), ref, bound, D)
    _check(head(_cuda(h)), ref, bound, D)
    # the rounding itself: 2^-4 of each factor at most (2^-4 + 2^-4 + 2^-8), and steps below the normal range
    exact = oracle.rms_norm(h.astype(np.float64), norm.astype(np.float64), 1e-5) @ lm_head.astype(np.float64)
    scale = np.abs(oracle.rms_norm(h.astype(np.float64), norm.astype(np.float64), 1e-5)) @ np.abs(lm_head)
    assert np.all(np.abs(head(h).cpu().numpy() - exact) <= 0.14 * scale)
    assert head(_cuda(h[:0])).shape == (0, V)
    w, x = head.weights, _cuda(h)
    with pytest.raises(TypeError):
        fp8_linear(x.double(), w)
    with pytest.raises(TypeError):
        fp8_linear(h, w)
    with pytest.raises(ValueError):
        fp8_linear(x[:, :255], w)
    with pytest.raises(ValueError):
        fp8_linear(torch.randn((D, 12), device="cuda").T, w)
    with pytest.raises(ValueError):
        fp8_linear(x, w, out=torch.empty((12, V + 1), device="cuda"))
    with pytest.raises(TypeError):
        fp8_linear(x, w, out=torch.empty((12, V), device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError):
        fp8_linear(x, w, out=torch.empty((1, V), device="cuda").expand(12, V))
    with pytest.raises(ValueError):
        fp8_linear(x, w, norm=head.norm[:-1])
    with pytest.raises(TypeError):
        fp8_linear(x, w, norm=head.norm.double())
    for eps in (float("nan"), -1.0):
        with pytest.raises(ValueError):
            fp8_linear(x, w, norm=head.norm, eps=eps)
    with pytest.raises(TypeError):
        Fp8Weights.quantize(np.zeros((4, 4)))
    with pytest.raises(ValueError):
        Fp8Weights.quantize(np.zeros(4, np.float32))
    with pytest.raises(ValueError):
        Fp8Weights.quantize(np.zeros((0, 4), np.float32))
    with pytest.raises(ValueError):
        Fp8Weights.from_codes(np.zeros((4, 4), np.uint8), np.ones((1, 2), np.float32))
    with pytest.raises(TypeError):
        Fp8Weights.from_codes(np.zeros((4, 4), np.int32), np.ones((1, 1), np.float32))
    with pytest.raises(TypeError):
        Fp8Weights.from_codes(np.zeros((4, 4), np.uint8), np.ones((1, 1)))


def test_refusals_of_the_library():
    import torch

    c = _native.Context(0)
    buf = torch.zeros(1 << 16, dtype=torch.uint8, device="cuda")
    p = buf.data_ptr()
    ok = [p, 0, 128, 4, 128, None, 1e-5, p, p, 64, p, 64, p, 1 << 16]
    assert c.fp8_ws_bytes(4, 64, 128) <= 1 << 16
    bad = [(0, None), (1, 1), (1, 4), (2, 127), (3, -1), (4, 0), (7, None), (7, p + 8), (8, None), (9, 0), (10, None),
           (10, p + 2), (11, 63), (12, None), (12, p + 128), (13, c.fp8_ws_bytes(4, 64, 128) - 1), (0, p + 2)]
    for i, v in bad:
        args = list(ok)
        args[i] = v
        with pytest.raises(ValueError):
            c.fp8_linear(*args)
    args = list(ok)
    args[5], args[6] = p, -1.0
    with pytest.raises(ValueError):
        c.fp8_linear(*args)
    for args in [(None, 128, p, 1, 64, 128, p, p), (p, 127, p, 1, 64, 128, p, p), (p, 128, p, 0, 64, 128, p, p),
                 (p, 128, p, 1, 0, 128, p, p), (p, 128, p, 1, 64, 128, p + 8, p)]:
        with pytest.raises(ValueError):
            c.fp8_pack(*args)
    for args in [(None, 0, 1, 64, 64, 128, p, p), (p, 1, 1, 64, 64, 128, p, p), (p, 0, -1, 64, 64, 128, p, p),
                 (p, 0, 1, 64, 64, 0, p, p), (p, 0, 1, 64, 64, 128, p + 4, p)]:
        with pytest.raises(ValueError):
            c.fp8_quantize(*args)
    c.close()


def test_offsets_past_32_bits():
    """More than 2^31 logits of 70001 rows, and rows of out that lie far apart."""
    import torch

    N, V, D = 70001, 31000, 128
    print("[fp8] 70001 x 31000", flush=True)
    g = np.random.default_rng(0)
    w = Fp8Weights.quantize(_cuda(_matrix(g, V, D)))
    x = torch.randn((N, D), device="cuda", dtype=torch.bfloat16)
    rows = [0, 65535, 65536, 69273, N - 1]
    ref, bound = O.linear(x[rows].double().cpu().numpy(), w.dequantize().double().cpu().numpy())
    out = fp8_linear(x, w)
    _check(out[rows], ref, bound, D)
    del out
    far = torch.zeros((3, 1 << 30), device="cuda")[:, 5:5 + V]
    fp8_linear(x[:3], w, out=far)
    ref, bound = O.linear(x[:3].double().cpu().numpy(), w.dequantize().double().cpu().numpy())
    _check(far, ref, bound, D)


def test_very_many_rows():
    """More rows than a grid has threads for, 512 each."""
    import torch

    N, D = 8_500_001, 16
    print("[fp8] 8500001 rows", flush=True)
    w = Fp8Weights.from_codes(_cuda(np.full((2, D), 0x38, dtype=np.uint8)), _cuda(np.array([[0.5]], dtype=np.float32)))
    x = torch.randn((N, D), device="cuda", dtype=torch.bfloat16)
    out = fp8_linear(x, w)
    rows = [0, (1 << 20) - 1, 1 << 20, 1 << 23, N - 1]
    ref, bound = O.linear(x[rows].double().cpu().numpy(), np.full((2, D), 0.5))
    _check(out[rows], ref, bound, D)
    # the rest: within e4m3's rounding of the float32 sums
    full = 0.5 * x.float().sum(1)
    assert bool(((out[:, 0] - full).abs() <= 0.5 * (2.0 ** -4 + 2.0 ** -9) * x.float().abs().sum(1) + 1e-6).all())


def test_refuses_more_codes_than_a_grid_holds():
    c = _native.Context(0)
    with pytest.raises(NotImplementedError):
        c.fp8_pack(256, 1 << 20, 256, 1 << 13, 1 << 16, 1 << 20, 256, 256)
    c.close()


def test_workspaces_of_very_many_rows():
    """The bytes of rows near 2^31 (nothing of that size is allocated), which no smaller
    workspace passes for; matrices past 2^35 codes are refused."""
    c = _native.Context(0)
    for N in (2**31 - 1, 2**31 - 31, 2**31 - 32, 2**31 - 200):
        assert c.fp8_ws_bytes(N, 1, 1) == -(-N // 32) * 32 * 128 * 2, N
        with pytest.raises(ValueError):  # before anything is launched: the pointers are never read
            c.fp8_linear(256, _native.PLH_BF16, 1, N, 1, None, 0.0, 256, 256, 1, 256, 1, 256, 1 << 38)
    assert c.fp8_ws_bytes(2**31 - 1, 32, 2**30) == 2**62
    assert c.fp8_ws_bytes(1, 2**31 - 1, 2**31 - 1) == _native.PLH_ERR_UNSUPPORTED
    assert c.fp8_ws_bytes(1, 2**29, 128) == _native.PLH_ERR_UNSUPPORTED
    c.close()


def test_sizes_past_int32_are_refused():
    """Not taken modulo 2^32 (nothing but the allocation happens at these sizes)."""
    import torch

    w = Fp8Weights.from_codes(np.zeros((1, 1), np.uint8), np.ones((1, 1), np.float32))
    print("[fp8] 2^32 + 10 rows", flush=True)
    x = torch.empty(2**32 + 10, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="2\\^31"):
        fp8_linear(x[:, None], w, out=torch.empty(1, device="cuda").expand(2**32 + 10, 1))
    for m in (x[:, None], x[None]):
        with pytest.raises(ValueError, match="2\\^31"):
            Fp8Weights.quantize(m)
