"""What lies between a step's last hidden states and its answer, beside sampling.

Each case is one pass through one operator on device-resident data:

  fp8       the final RMSNorm and the lm_head product with e4m3 weights, one
            float32 scale for each 128 x 128 block of them, and the rows
            rounded to e4m3 with a scale for each 128 of a row
  process   biases, repetition, frequency and presence penalties and grammar
            masks on a batch's logits
  logprobs  the log probability and rank of each row's chosen token, and the
            row's best tokens with theirs

`run` computes them from elementary torch operations, or with `own` set by
this package's kernels.
"""

from __future__ import annotations

import math

import torch

own = False

BLOCK = 128
E4M3_MAX = 448.0


def listed() -> list[dict]:
    return [
        # the logits of a few interactive requests over a 128k vocabulary
        dict(name="fp8_8x128k", kind="fp8", rows=8, vocab=128256, width=4096, dtype="float32"),
        # the logits of a full batch
        dict(name="fp8_256x128k", kind="fp8", rows=256, vocab=128256, width=4096, dtype="bfloat16"),
        # an odd vocabulary and width, and a batch between the two
        dict(name="fp8_45x50k", kind="fp8", rows=45, vocab=50257, width=1000, dtype="float16"),
        # the logits at every position of a prompt, to score it
        dict(name="fp8_prompt32k", kind="fp8", rows=2048, vocab=32000, width=4096, dtype="bfloat16"),
        # a character-level model's step: the smallest call
        dict(name="process_char", kind="process", rows=16, vocab=65, dtype="float32", mode="chat", hist=64, bias=4),
        # chat requests of a 32k-token model: penalties and a few biased tokens
        dict(name="process_chat32k", kind="process", rows=64, vocab=32000, dtype="float32", mode="chat", hist=512,
             bias=32),
        # 256 requests of four kinds: plain ones, penalties, a grammar, both
        dict(name="process_mixed128k", kind="process", rows=256, vocab=128256, dtype="float32", mode="mixed",
             hist=2048, bias=64),
        # float64 logits of an odd vocabulary, every request under a grammar, long histories
        dict(name="process_f64_50k", kind="process", rows=32, vocab=50257, dtype="float64", mode="grammar", hist=4096,
             bias=300),
        # a character-level model's answer
        dict(name="logprobs_char", kind="logprobs", rows=16, vocab=65, dtype="float32", top=5),
        # a full batch whose requests ask for the twenty best tokens
        dict(name="logprobs_256x128k", kind="logprobs", rows=256, vocab=128256, dtype="float32", top=20),
        # a prompt's own tokens, scored
        dict(name="logprobs_prompt32k", kind="logprobs", rows=2048, vocab=32000, dtype="float32", top=0),
        # float64 logits of an odd vocabulary
        dict(name="logprobs_f64_50k", kind="logprobs", rows=48, vocab=50257, dtype="float64", top=20),
    ]


_MOST_MACS = 256 * 4096 * 128256
_MOST_ELEMENTS = 256 * 128256


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["fp8", "process", "logprobs"])
    if kind == "fp8":
        c = dict(kind=kind, rows=_log_int(rng, 1, 2048), vocab=_log_int(rng, 65, 128256), width=_log_int(rng, 64, 4096),
                 dtype=rng.choice(["float32", "bfloat16", "float16"]))
        if rng.random() < 0.5:  # sizes as models have them, in whole blocks
            c["vocab"], c["width"] = min(-(-c["vocab"] // 128) * 128, 128256), -(-c["width"] // 128) * 128
        c["rows"] = max(1, min(c["rows"], _MOST_MACS // (c["vocab"] * c["width"])))
        return c
    c = dict(kind=kind, rows=_log_int(rng, 1, 256 if kind == "process" else 2048), vocab=_log_int(rng, 65, 152064),
             dtype=rng.choice(["float32", "float32", "float32", "float64"]))
    most = _MOST_ELEMENTS if c["dtype"] == "float32" else _MOST_ELEMENTS // 2
    c["rows"] = max(1, min(c["rows"], most // c["vocab"]))
    if kind == "process":
        c["mode"] = rng.choice(["chat", "mixed", "grammar"])
        c["hist"] = rng.choice([0, _log_int(rng, 1, 4096), _log_int(rng, 1, 4096), _log_int(rng, 1, 4096)])
        c["bias"] = min(rng.choice([0, _log_int(rng, 1, 300)]), c["vocab"] // 2)
    else:
        c["top"] = rng.choice([0, 1, 5, 20, rng.randint(1, 64)])
    return c


# ------------------------------------------------------------------- inputs


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) % (1 << 62))
    return g


def _quantised_weights(g, V: int, D: int):
    """(codes [V, D] float8_e4m3fn, scales [V/128, D/128] float32) of normal
    weights whose size differs from block to block, as a checkpoint holds them."""
    vb, db = -(-V // BLOCK), -(-D // BLOCK)
    spread = torch.exp2(1.5 * torch.randn((vb, db), generator=g, device="cuda"))
    codes = torch.empty((V, D), dtype=torch.float8_e4m3fn, device="cuda")
    scales = torch.empty((vb, db), dtype=torch.float32, device="cuda")
    for b in range(0, vb, 128):  # 16384 rows at a time
        v0, v1 = b * BLOCK, min(V, (b + 128) * BLOCK)
        n = -(-(v1 - v0) // BLOCK)
        w = torch.zeros((n * BLOCK, db * BLOCK), device="cuda")
        w[:v1 - v0, :D] = torch.randn((v1 - v0, D), generator=g, device="cuda").mul_(0.02)
        w = w.view(n, BLOCK, db, BLOCK) * spread[b:b + n, None, :, None]
        s = w.abs().amax((1, 3)) / E4M3_MAX
        scales[b:b + n] = s
        q = (w / s[:, None, :, None]).clamp_(-E4M3_MAX, E4M3_MAX).view(n * BLOCK, db * BLOCK)
        codes[v0:v1] = q[:v1 - v0, :D].to(torch.float8_e4m3fn)
    return codes, scales


def _fp8_inputs(case: dict, seed: int):
    g = _gen(seed)
    N, D, V = case["rows"], case["width"], case["vocab"]
    h = torch.randn((N, D), generator=g, device="cuda").to(getattr(torch, case["dtype"]))
    norm = 1 + 0.1 * torch.randn(D, generator=g, device="cuda")
    codes, scales = _quantised_weights(g, V, D)
    return h, norm, codes, scales


# (repetition, frequency, presence penalty, under a grammar) of a batch's rows
_KINDS = {
    "chat": [(1.1, 0.5, 0.25, False), (1.0, 0.7, 0.0, False), (1.2, 0.0, 0.4, False)],
    "mixed": [(1.0, 0.0, 0.0, False), (1.1, 0.5, 0.25, False), (1.0, 0.0, 0.0, True), (1.05, 0.2, 0.1, True)],
    "grammar": [(1.05, 0.2, 0.1, True), (1.0, 0.0, 0.0, True)],
}


def _process_inputs(case: dict, seed: int) -> dict:
    g = _gen(seed)
    B, V, H, nb = case["rows"], case["vocab"], case["hist"], case["bias"]
    dt = getattr(torch, case["dtype"])
    kinds = [_KINDS[case["mode"]][b % len(_KINDS[case["mode"]])] for b in range(B)]
    col = lambda i: torch.tensor([k[i] for k in kinds], dtype=torch.float64, device="cuda")  # noqa: E731
    d = dict(x=3.0 * torch.randn((B, V), generator=g, device="cuda", dtype=dt), rep=col(0), freq=col(1), pres=col(2))
    # histories that repeat themselves: ranks from a power law, scattered over
    # the vocabulary, of lengths between half of H and H; the last third is output
    lens = torch.randint(H // 2, H + 1, (B,), generator=g, device="cuda") if H else torch.zeros(B, device="cuda").long()
    d["hist_off"] = torch.cat([torch.zeros(1, dtype=torch.int64, device="cuda"), lens.cumsum(0)])
    d["total"] = int(d["hist_off"][-1])
    u = torch.rand(d["total"], generator=g, device="cuda", dtype=torch.float64)
    d["hist_ids"] = (((V ** u).long() - 1) * 7919 % V).to(torch.int32)
    d["out_start"] = 2 * lens // 3
    # each row's biased tokens, ascending
    ids = torch.rand((B, V), generator=g, device="cuda").topk(nb, dim=1).indices.sort(1).values
    d["bias_ids"] = ids.to(torch.int32).reshape(-1)
    d["bias"] = 2.0 * torch.randn(B * nb, generator=g, device="cuda", dtype=torch.float64)
    d["bias_off"] = nb * torch.arange(B + 1, device="cuda")
    # bitmasks of the rows under a grammar: from a few tokens allowed to nearly all
    row = [-1] * B
    for b, r in enumerate(b for b in range(B) if kinds[b][3]):
        row[r] = b
    M, words = max(1, max(row) + 1), -(-V // 32)
    share = torch.rand((M, 1), generator=g, device="cuda") ** 4
    bits = torch.rand((M, words * 32), generator=g, device="cuda") < share
    bits = bits.view(M, words, 32).long() << torch.arange(32, device="cuda")
    d["mask"] = bits.sum(-1).to(torch.int32)  # two's complement of the unsigned words
    d["mask_row"] = torch.tensor(row, dtype=torch.int32, device="cuda")
    return d


def _logprobs_inputs(case: dict, seed: int):
    """Logits with a few likely tokens and, in every other row, a tenth of
    the tokens ruled out; the chosen token is among the likelier ones."""
    g = _gen(seed)
    B, V = case["rows"], case["vocab"]
    x = 3.0 * torch.randn((B, V), generator=g, device="cuda", dtype=getattr(torch, case["dtype"]))
    n = min(8, V)
    top = torch.rand((B, V), generator=g, device="cuda").topk(n, dim=1).indices
    x.scatter_(1, top, 10.0 + 3.0 * torch.randn((B, n), generator=g, device="cuda", dtype=x.dtype))
    for b in range(0, B, 512):  # every other row, 512 rows at a time
        part = x[b + 1:b + 512:2]
        part.masked_fill_(torch.rand(part.shape, generator=g, device="cuda") < 0.1, -math.inf)
    pick = torch.randint(0, n, (B,), generator=g, device="cuda")
    return x, top.gather(1, pick[:, None])[:, 0].to(torch.int32)


def prepare(case: dict, seed: int) -> dict:
    s = dict(kind=case["kind"], case=case)
    if case["kind"] == "fp8":
        s["h"], s["norm"], s["codes"], s["scales"] = _fp8_inputs(case, seed)
        s["out"] = torch.empty((case["rows"], case["vocab"]), device="cuda")
        if own:  # the weights as a server keeps them, laid out once when they are loaded
            from pagellm_amd.fp8 import Fp8LogitsHead

            s["head"] = Fp8LogitsHead.from_codes(s["norm"], s["codes"], s["scales"], 1e-5)
        return s
    if case["kind"] == "process":
        s.update(_process_inputs(case, seed))
        s["out"] = torch.empty_like(s["x"])
    else:
        s["x"], s["ids"] = _logprobs_inputs(case, seed)
        B, n = case["rows"], case["top"]
        s["lp"], s["rank"] = torch.empty(B, dtype=s["x"].dtype, device="cuda"), torch.empty_like(s["ids"])
        s["top_ids"] = torch.empty((B, n), dtype=torch.int32, device="cuda")
        s["top_lp"] = torch.empty((B, n), dtype=s["x"].dtype, device="cuda")
    if own:
        from pagellm_amd import _native

        s["ctx"], s["dtype"] = _native.default_context(), _native.dtype_code(case["dtype"])
    return s


# -------------------------------------------------------------- plain forms


def _fp8_plain(h, norm, codes, scales):
    (N, D), V = h.shape, codes.shape[0]
    db = -(-D // BLOCK)
    h = h.double()  # a value next to a border between two codes
    y = (h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5) * norm.double()).float()
    y = torch.nn.functional.pad(y, (0, db * BLOCK - D)).view(N, db, BLOCK)
    # the smallest power of two s with max|y| <= 448 s
    m, e = torch.frexp(y.abs().amax(-1, keepdim=True))
    s = torch.ldexp(torch.ones_like(m), torch.where(m > 0.875, e - 8, e - 9).clamp_min(-126))
    a = ((y / s).to(torch.float8_e4m3fn).float() * s).view(N, db * BLOCK)[:, :D]
    t = scales.repeat_interleave(BLOCK, 0)[:V].repeat_interleave(BLOCK, 1)[:, :D]
    return a @ (codes.float() * t).T


def _process_plain(s: dict):
    x = s["x"]
    (B, V), dt = x.shape, x.dtype
    rows = torch.arange(B, device="cuda")
    y = x
    if s["bias"].numel():
        bias = torch.zeros_like(x)
        at = torch.repeat_interleave(rows, s["bias_off"].diff(), output_size=s["bias"].numel())
        bias[at, s["bias_ids"].long()] = s["bias"].to(dt)
        y = y + bias
    if s["total"]:
        at = torch.repeat_interleave(rows, s["hist_off"].diff(), output_size=s["total"])
        ids = s["hist_ids"].long()
        seen = torch.zeros((B, V), dtype=torch.bool, device="cuda")
        seen[at, ids] = True
        r = s["rep"].to(dt)[:, None]
        y = torch.where(seen, torch.where(y > 0, y / r, y * r), y)
        is_output = torch.arange(s["total"], device="cuda") - s["hist_off"][at] >= s["out_start"][at]
        count = torch.zeros_like(x).index_put_((at, ids), is_output.to(dt), accumulate=True)
        y = y - (s["freq"].to(dt)[:, None] * count + s["pres"].to(dt)[:, None] * (count > 0))
    words = s["mask"][s["mask_row"].clamp_min(0).long()]
    tokens = torch.arange(V, device="cuda")
    allowed = (words[:, tokens // 32] >> (tokens % 32)) & 1 != 0
    return torch.where(allowed | (s["mask_row"] < 0)[:, None], y, -math.inf)


def _order_key(x):
    """Keys that sort as the values do, in the sign-magnitude order of IEEE floats."""
    i = (x + 0.0).view(torch.int32 if x.dtype == torch.float32 else torch.int64).long()
    return torch.where(i < 0, i ^ (0x7FFFFFFF if x.dtype == torch.float32 else 0x7FFFFFFFFFFFFFFF), i)


def _logprobs_plain(x, ids, n: int):
    B, V = x.shape
    m = x.amax(1, keepdim=True)
    lse = m + torch.log(torch.exp(x - m).sum(1, keepdim=True))
    chosen = x.gather(1, ids.long()[:, None])
    tokens = torch.arange(V, device="cuda")
    rank = 1 + ((x > chosen) | ((x == chosen) & (tokens < ids[:, None]))).sum(1)
    if x.dtype == torch.float32:  # value, then the lower token, in one integer
        top = torch.topk((_order_key(x) << 32) - tokens, n, dim=1).indices
    else:
        top = torch.sort(_order_key(x), dim=1, descending=True, stable=True).indices[:, :n]
    return (chosen - lse)[:, 0], rank.to(torch.int32), top.to(torch.int32), x.gather(1, top) - lse


def run(s: dict):
    kind, case = s["kind"], s["case"]
    if not own:
        if kind == "fp8":
            return _fp8_plain(s["h"], s["norm"], s["codes"], s["scales"])
        return _process_plain(s) if kind == "process" else _logprobs_plain(s["x"], s["ids"], case["top"])
    if kind == "fp8":
        return s["head"](s["h"], out=s["out"])
    B, V, c = case["rows"], case["vocab"], s["ctx"]
    c.set_stream(torch.cuda.current_stream().cuda_stream)
    if kind == "process":
        at = lambda name, by: s[name].data_ptr() if s[by].numel() else None  # noqa: E731
        c.process_logits(s["x"].data_ptr(), s["dtype"], V, B, V, at("hist_ids", "hist_ids"),
                         at("hist_off", "hist_ids"), at("out_start", "hist_ids"), s["rep"].data_ptr(),
                         s["freq"].data_ptr(), s["pres"].data_ptr(), at("bias_ids", "bias"), at("bias", "bias"),
                         at("bias_off", "bias"), s["mask"].data_ptr(), s["mask"].shape[1], s["mask"].shape[0],
                         s["mask_row"].data_ptr(), s["out"].data_ptr(), V)
        return s["out"]
    c.logprobs(s["x"].data_ptr(), s["dtype"], V, B, V, s["ids"].data_ptr(), s["lp"].data_ptr(), s["rank"].data_ptr(),
               case["top"], s["top_ids"].data_ptr(), s["top_lp"].data_ptr())
    return s["lp"], s["rank"], s["top_ids"], s["top_lp"]


def work(case: dict) -> dict:
    B, V = case["rows"], case["vocab"]
    e = {"float64": 8, "float32": 4}.get(case["dtype"], 2)
    if case["kind"] == "fp8":
        D = case["width"]
        blocks = -(-V // BLOCK) * -(-D // BLOCK)
        return {"bytes": V * D + 4 * blocks + e * B * D + 4 * D + 4 * B * V, "flops": 2 * B * D * V}
    if case["kind"] == "process":
        masked = sum(_KINDS[case["mode"]][b % len(_KINDS[case["mode"]])][3] for b in range(B))
        rows = 2 * e * V + 3 * case["hist"] + 12 * case["bias"] + 52  # histories are three quarters of hist long
        return {"bytes": B * rows + masked * V // 8, "flops": B * V}
    return {"bytes": B * (e * V + (e + 4) * case["top"] + e + 8), "flops": 4 * B * V}


# ------------------------------------------------- the same in plain float64


def _fp8_exact(h, norm, codes, scales):
    (N, D), V = h.shape, codes.shape[0]
    x = h.double()
    y = ((x * torch.rsqrt(x.square().sum(1) / D + 1e-5)[:, None]) * norm.double()).float().double()
    a = torch.empty_like(y)
    for k in range(0, D, BLOCK):
        part = y[:, k:k + BLOCK]
        big = part.abs().amax(1, keepdim=True).clamp_min(2.0 ** -110)
        s = 2.0 ** torch.ceil(torch.log2(big / E4M3_MAX))
        s = torch.where(big <= E4M3_MAX * s / 2, s / 2, torch.where(big > E4M3_MAX * s, 2 * s, s))
        # e4m3: steps of 2^-3 of the value's power of two, of 2^-9 below 2^-6
        q = part / s
        step = 2.0 ** (torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
        a[:, k:k + BLOCK] = torch.round(q / step) * step * s  # to even
    out = torch.empty((N, V), dtype=torch.float64, device="cuda")
    for v in range(0, V, 8192):
        w = codes[v:v + 8192].double()
        at = torch.arange(v, v + w.shape[0], device="cuda") // BLOCK
        w *= scales.double()[at][:, torch.arange(D, device="cuda") // BLOCK]
        out[:, v:v + 8192] = a @ w.T.contiguous()
    return out


def _process_exact(d: dict):
    out = d["x"].double().clone()
    V = out.shape[1]
    off, start, b_off = d["hist_off"].tolist(), d["out_start"].tolist(), d["bias_off"].tolist()
    rep, freq, pres, mask_row = d["rep"].tolist(), d["freq"].tolist(), d["pres"].tolist(), d["mask_row"].tolist()
    for b in range(out.shape[0]):
        y = out[b]
        y[d["bias_ids"][b_off[b]:b_off[b + 1]].long()] += d["bias"][b_off[b]:b_off[b + 1]]
        hist = d["hist_ids"][off[b]:off[b + 1]].long()
        if hist.numel():
            t = hist.unique()
            y[t] = torch.where(y[t] > 0, y[t] / rep[b], y[t] * rep[b])
            t, n = hist[start[b]:].unique(return_counts=True)
            y[t] -= freq[b] * n.double() + pres[b]
        if mask_row[b] >= 0:
            words = d["mask"][mask_row[b]]
            bits = torch.stack([(words >> i) & 1 for i in range(32)], dim=1).reshape(-1)[:V]
            y[bits == 0] = -math.inf
    return out


def _logprobs_exact(x, ids, n: int):
    x = x.double()
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    rank = (order == ids[:, None]).long().argmax(1) + 1
    lp = torch.log_softmax(x, dim=1)
    top = order[:, :n]
    return lp.gather(1, ids.long()[:, None])[:, 0], rank.to(torch.int32), top.to(torch.int32), lp.gather(1, top)


def exact(case: dict, seed: int):
    """What run() returns, in plain float64."""
    if case["kind"] == "fp8":
        return _fp8_exact(*_fp8_inputs(case, seed))
    if case["kind"] == "process":
        return _process_exact(_process_inputs(case, seed))
    return _logprobs_exact(*_logprobs_inputs(case, seed), case["top"])
