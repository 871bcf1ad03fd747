"""One round of speculation with trees of drafted tokens, on the target's side.

Each case is one pass through one operator on device-resident data:

  attend   attention of each sequence's tree nodes (one node: single-token
           decoding; width 1: a chain of tokens) over its pages of a key and
           value cache
  rotary   rotary positions of queries and keys, keys and values written into
           their places in the cache
  verify   the accepted path of each sequence's tree and the token after it,
           from given uniforms
  copy     pages of all layers copied, as forked sequences need them
  keep     the accepted nodes' keys and values of all layers moved together

`run` computes them from elementary torch operations, or with `own` set by
this package's kernels.
"""

from __future__ import annotations

import math

import torch

own = False


def listed() -> list[dict]:
    return [
        # a character-level float32 model that verifies chains of four drafts
        dict(name="attend_char", kind="attend", batch=16, nodes=5, width=1, heads=6, kv_heads=6, dim=64, page=16,
             length=256, dtype="float32"),
        # a full batch decodes one token each over contexts of up to 8192
        dict(name="attend_decode", kind="attend", batch=64, nodes=1, width=1, heads=32, kv_heads=8, dim=128, page=16,
             length=8192, dtype="bfloat16"),
        # binary trees of up to 32 drafts
        dict(name="attend_tree32", kind="attend", batch=32, nodes=32, width=2, heads=32, kv_heads=8, dim=128, page=32,
             length=4096, dtype="bfloat16"),
        # the largest trees over long contexts, for few sequences
        dict(name="attend_tree64_long", kind="attend", batch=4, nodes=64, width=4, heads=64, kv_heads=8, dim=128,
             page=64, length=32768, dtype="float16"),
        # a decode step's rows
        dict(name="rotary_step", kind="rotary", tokens=64, heads=32, kv_heads=8, dim=128, part=128, layout="half",
             scaling="none", page=16, last=8192, dtype="bfloat16"),
        # a long prompt's rows at far positions: interleaved pairs in half of the head, frequencies stretched
        dict(name="rotary_prompt", kind="rotary", tokens=8192, heads=32, kv_heads=8, dim=128, part=64,
             layout="interleaved", scaling="yarn", page=16, last=131072, dtype="float16"),
        # a batch of binary trees, distributions as the sampler exports them
        dict(name="verify_32k", kind="verify", batch=64, nodes=16, width=2, vocab=32000, dtype="float64",
             replacement=False),
        # few sequences with wide trees over a 128k vocabulary
        dict(name="verify_128k", kind="verify", batch=8, nodes=32, width=4, vocab=128256, dtype="float32",
             replacement=False),
        # a few requests fork: the last page of each is copied
        dict(name="copy_fork", kind="copy", pairs=8, pages=64, layers=16, kv_heads=8, dim=128, page=16,
             dtype="bfloat16"),
        # the pages of a large batch moved together
        dict(name="copy_many", kind="copy", pairs=512, pages=1152, layers=16, kv_heads=8, dim=128, page=16,
             dtype="bfloat16"),
        # the accepted drafts of a small batch
        dict(name="keep_step", kind="keep", batch=8, nodes=16, layers=16, kv_heads=8, dim=128, page=16, length=256,
             dtype="bfloat16"),
        # the accepted drafts of a full batch with the largest trees
        dict(name="keep_batch", kind="keep", batch=64, nodes=64, layers=32, kv_heads=8, dim=128, page=16, length=256,
             dtype="bfloat16"),
    ]


_BYTES = {"float64": 8, "float32": 4, "bfloat16": 2, "float16": 2}
_MOST_CACHE = 64 * 8192 * 8 * 128 * 2  # bytes of keys of one layer
_MOST_PRODUCTS = 4 * 64 * 64 * 32768 * 128
_MOST_PROBS = 64 * 16 * 32000 * 8
_MOST_POOL = 1152 * 16 * 8 * 16 * 128 * 2


def _log_int(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["attend", "attend", "attend", "rotary", "verify", "verify", "copy", "keep"])
    if kind == "verify":
        c = dict(kind=kind, batch=_log_int(rng, 1, 128), width=rng.choice([1, 2, 3, 4, 8]), vocab=_log_int(rng, 65, 152064),
                 dtype=rng.choice(["float32", "float64"]), replacement=rng.random() < 0.25)
        c["nodes"] = _log_int(rng, 1, 64)
        c["batch"] = max(1, min(c["batch"], _MOST_PROBS // (_BYTES[c["dtype"]] * c["vocab"] * c["nodes"])))
        return c
    c = dict(kind=kind, kv_heads=rng.choice([1, 2, 4, 6, 8]), dim=rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 256]),
             page=rng.choice([16, 16, 32, 64, 128]), dtype=rng.choice(["bfloat16", "bfloat16", "float16", "float32"]))
    e = _BYTES[c["dtype"]]
    if kind == "attend":
        c["heads"] = c["kv_heads"] * rng.choice([1, 2, 4, 7, 8])
        c["width"] = rng.choice([1, 1, 2, 3, 4])
        c["nodes"] = _log_int(rng, 1, 64) if c["width"] > 1 else rng.choice([1, 1, _log_int(rng, 2, 300)])
        c["length"] = _log_int(rng, 1, 65536)
        c["batch"] = _log_int(rng, 1, 128)
        key = c["kv_heads"] * c["dim"] * e
        c["length"] = min(c["length"], _MOST_CACHE // key)
        c["nodes"] = max(1, min(c["nodes"], _MOST_PRODUCTS // (8 * c["heads"] * c["dim"] * (c["length"] + c["nodes"]))))
        c["batch"] = max(1, min(c["batch"], _MOST_CACHE // (key * (c["length"] + c["nodes"])),
                                _MOST_PRODUCTS // (8 * c["nodes"] * c["heads"] * c["dim"] * (c["length"] + c["nodes"]))))
    elif kind == "rotary":
        c.update(tokens=_log_int(rng, 1, 8192), heads=c["kv_heads"] * rng.choice([1, 2, 4, 7]),
                 part=rng.choice([c["dim"], c["dim"], c["dim"] // 2, c["dim"] // 4]),
                 layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "yarn"]),
                 last=_log_int(rng, 64, 1048576))
        c["tokens"] = max(1, min(c["tokens"], 8192 * 48 * 128 * 2 // ((c["heads"] + 2 * c["kv_heads"]) * c["dim"] * e)))
    else:
        c["layers"] = rng.randint(1, 32)
        page = c["layers"] * c["kv_heads"] * c["dim"] * c["page"] * e  # of keys
        if kind == "copy":
            c["pairs"] = max(1, min(_log_int(rng, 1, 512), _MOST_POOL * 4 // 9 // page))
            c["pages"] = 2 * c["pairs"] + rng.randint(0, c["pairs"])
        else:
            c.update(batch=_log_int(rng, 1, 64), nodes=_log_int(rng, 1, 64), length=_log_int(rng, 1, 1000))
            c["batch"] = max(1, min(c["batch"], _MOST_POOL // (page * _pages_each(c))))
    return c


def _pages_each(c: dict) -> int:
    return -(-(c["length"] + c["nodes"]) // c["page"])


# ------------------------------------------------------------------- inputs


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) % (1 << 62))
    return g


def _node_counts(B: int, T: int):
    """Nodes of each sequence's tree, from half of T to T (the first T; the
    same for every seed), and of all rows: their offsets, each row's sequence
    and its place there."""
    n = T - torch.arange(B, device="cuda") * 5 % (T // 2 + 1)
    off = torch.cat([n.new_zeros(1), n.cumsum(0)])
    seq = torch.repeat_interleave(torch.arange(B, device="cuda"), n)
    return n, off, seq, torch.arange(seq.numel(), device="cuda") - off[seq]


def _tree_parents(T: int, width: int) -> list[int]:
    """Level by level, each node with `width` children."""
    return [-1] + [(i - 1) // width for i in range(1, T)]


def _paged_table(g, B: int, each: int):
    """Page numbers [B, each], scattered over the pool."""
    return torch.randperm(B * each, generator=g, device="cuda").view(B, each).to(torch.int32)


def _attend_inputs(c: dict, seed: int) -> dict:
    g = _gen(seed)
    B, T, Hq, Hkv, D = c["batch"], c["nodes"], c["heads"], c["kv_heads"], c["dim"]
    dt = getattr(torch, c["dtype"])
    _, off, seq, place = _node_counts(B, T)
    lens = torch.randint(c["length"] // 2, c["length"] + 1, (B,), generator=g, device="cuda")
    lens[0] = c["length"]
    each = _pages_each(c)
    pool = (B * each, Hkv, c["page"], D)
    d = dict(node_off=off.to(torch.int32), lens=lens.to(torch.int32), table=_paged_table(g, B, each), seq=seq, place=place)
    d["k"] = torch.randn(pool, generator=g, device="cuda", dtype=dt)
    d["v"] = torch.randn(pool, generator=g, device="cuda", dtype=dt)
    d["q"] = torch.randn((seq.numel(), Hq, D), generator=g, device="cuda", dtype=dt) * 1.5
    d["visible"] = None
    if c["width"] > 1:  # each node sees its ancestors and itself
        bits = []
        for i, p in enumerate(_tree_parents(T, c["width"])):
            bits.append((bits[p] if i else 0) | 1 << i)
        bits = torch.tensor([b - (1 << 64) if b >= 1 << 63 else b for b in bits], device="cuda")
        d["visible"] = bits[place]
    return d


def _frequencies(c: dict):
    """(radians a position [part / 2] in float64, factor on the rotated values)"""
    i = torch.arange(c["part"] // 2, dtype=torch.float64, device="cuda")
    f = 10000.0 ** (-2.0 * i / c["part"])
    if c["scaling"] == "linear":
        return f / 8.0, 1.0
    if c["scaling"] == "yarn":  # slow pairs stretched by 16, fast ones as they are, a ramp between the two
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        return f * keep + f / 16.0 * (1.0 - keep), 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def _rotary_inputs(c: dict, seed: int) -> dict:
    g = _gen(seed)
    N, Hq, Hkv, D, ps = c["tokens"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    dt = getattr(torch, c["dtype"])
    pages = -(-N // ps) + 8
    d = dict(qkv=torch.randn((N, (Hq + 2 * Hkv) * D), generator=g, device="cuda", dtype=dt))
    d["pos"] = torch.randint(0, c["last"], (N,), generator=g, device="cuda")
    d["slots"] = torch.randperm(pages * ps, generator=g, device="cuda")[:N]
    d["k"] = torch.randn((pages, Hkv, ps, D), generator=g, device="cuda", dtype=dt)
    d["v"] = torch.randn((pages, Hkv, ps, D), generator=g, device="cuda", dtype=dt)
    d["freq"], d["factor"] = _frequencies(c)
    return d


def _verify_inputs(c: dict, seed: int) -> dict:
    """Peaked target distributions, the draft's near to them, and each node's
    children drawn from the draft's, mostly without replacement."""
    g = _gen(seed)
    B, T, V, w = c["batch"], c["nodes"], c["vocab"], c["width"]
    dt = getattr(torch, c["dtype"])
    _, off, seq, place = _node_counts(B, T)
    N = seq.numel()
    p = torch.empty((N, V), dtype=dt, device="cuda")
    q = torch.empty((N, V), dtype=dt, device="cuda")
    kids = torch.empty((N, w), dtype=torch.int64, device="cuda")
    for a in range(0, N, 128):  # 128 rows at a time
        n = min(128, N - a)
        z = 2.0 * torch.randn((n, V), generator=g, device="cuda")
        z.scatter_add_(1, torch.randint(0, V, (n, 12), generator=g, device="cuda"), torch.full((n, 12), 9.0, device="cuda"))
        zq = 0.7 * z + 1.2 * torch.randn((n, V), generator=g, device="cuda")
        p[a:a + n], q[a:a + n] = torch.softmax(z.to(dt), 1), torch.softmax(zq.to(dt), 1)
        if c["replacement"]:
            kids[a:a + n] = torch.multinomial(q[a:a + n].float(), w, replacement=True, generator=g)
        else:
            noise = -torch.log(torch.empty_like(zq).exponential_(generator=g))
            kids[a:a + n] = (zq + noise).topk(w, dim=1).indices
    parents = torch.tensor(_tree_parents(T, w), device="cuda")[place]
    which = (place - 1) % w  # of the parent's children
    tokens = kids[(off[seq] + parents).clamp_min(0), which]
    return dict(p=p, q=q, tokens=tokens.to(torch.int32), parents=parents.to(torch.int32), node_off=off.to(torch.int32),
                u=torch.rand((B, T), generator=g, device="cuda", dtype=torch.float64))


def _copy_inputs(c: dict, seed: int) -> dict:
    g = _gen(seed)
    pool = (c["layers"], c["pages"], c["kv_heads"], c["page"], c["dim"])
    dt = getattr(torch, c["dtype"])
    at = torch.randperm(c["pages"], generator=g, device="cuda")[:2 * c["pairs"]].to(torch.int32)
    return dict(k=torch.randn(pool, generator=g, device="cuda", dtype=dt), src=at[:c["pairs"]].contiguous(),
                v=torch.randn(pool, generator=g, device="cuda", dtype=dt), dst=at[c["pairs"]:].contiguous())


def _keep_inputs(c: dict, seed: int) -> dict:
    """Accepted nodes are a tree's first ones, or lie behind the places that
    the accepted ones move to (so that a second pass moves the same values)."""
    g = _gen(seed)
    B, T = c["batch"], c["nodes"]
    each = _pages_each(c)
    pool = (c["layers"], B * each, c["kv_heads"], c["page"], c["dim"])
    dt = getattr(torch, c["dtype"])
    d = dict(k=torch.randn(pool, generator=g, device="cuda", dtype=dt), table=_paged_table(g, B, each),
             v=torch.randn(pool, generator=g, device="cuda", dtype=dt))
    d["lens"] = torch.randint(0, c["length"] + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    n = torch.randint(0, min(8, T), (B,), generator=g, device="cuda")
    own_place = torch.randint(0, 3, (B,), generator=g, device="cuda")  # nodes that stay where they are
    j = torch.arange(T, device="cuda")
    key = torch.rand((B, T), generator=g, device="cuda")
    first = torch.minimum(own_place, n)[:, None]
    key = torch.where(j <= first, j - T - 1.0, torch.where(j <= n[:, None], 2.0, key))
    order = key.sort(1).indices  # 0 .. first, then nodes past n in any order, then the others
    path = torch.where(j <= n[:, None], order, T).sort(1).values
    n = torch.minimum(n, first[:, 0] + (T - 1 - n))  # as many as there are
    d["path"] = torch.where(j <= n[:, None], path, -1).to(torch.int32)
    d["n"] = n.to(torch.int32)
    return d


_INPUTS = {"attend": _attend_inputs, "rotary": _rotary_inputs, "verify": _verify_inputs, "copy": _copy_inputs,
           "keep": _keep_inputs}


def prepare(case: dict, seed: int) -> dict:
    s = _INPUTS[case["kind"]](case, seed)
    s["case"] = case
    if case["kind"] == "attend":
        s["out"] = torch.empty_like(s["q"])
    if case["kind"] == "rotary":
        N, D = case["tokens"], case["dim"]
        s["out"] = torch.empty((N, case["heads"], D), dtype=s["qkv"].dtype, device="cuda")
        if own:
            from pagellm_amd.cache import Rotary

            s["rotary"] = Rotary(inv_freq=s["freq"], layout=case["layout"], factor=s["factor"])
    return s


# -------------------------------------------------------------- plain forms


def _attend_plain(s: dict):
    c = s["case"]
    B, T, Hq, Hkv, D, ps = c["batch"], c["nodes"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    G = Hq // Hkv
    at = torch.arange(c["length"] + T, device="cuda")
    page = s["table"].long()[:, at // ps]
    keys, values = (s[n][page, :, at % ps].float() for n in ("k", "v"))  # [B, L, Hkv, D]
    seq, place, lens = s["seq"], s["place"], s["lens"].long()
    q = torch.zeros((B, T, Hq, D), device="cuda")
    q[seq, place] = s["q"].float()
    q = q.view(B, T, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, T * G, D)
    x = q @ keys.permute(0, 2, 3, 1).contiguous() * D ** -0.5
    node = at - lens[:, None]  # [B, L]: the tree's nodes from 0 on
    row = torch.arange(T, device="cuda")[None, :, None]
    if s["visible"] is None:
        sees = node[:, None] <= row
    else:
        bits = torch.zeros((B, T), dtype=torch.int64, device="cuda")
        bits[seq, place] = s["visible"]
        seen = (bits[:, :, None] >> node[:, None].clamp(0, 63)) & 1 != 0
        sees = (node[:, None] < 0) | (seen & (node[:, None] < 64))
    x = torch.where(sees.repeat_interleave(G, 1)[:, None], x, -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True).clamp_min(-1e30))
    o = (x @ values.permute(0, 2, 1, 3).contiguous()) / x.sum(-1, keepdim=True).clamp_min(1e-30)
    o = o.view(B, Hkv, T, G, D).permute(0, 2, 1, 3, 4).reshape(B, T, Hq, D)
    return o[seq, place].to(s["q"].dtype)


def _rotate(x, cos, sin, layout: str):
    """Pairs of the first 2 * cos.shape[1] values of each head turned."""
    R = 2 * cos.shape[1]
    part, rest = x[..., :R], x[..., R:]
    cos, sin = cos[:, None], sin[:, None]
    if layout == "half":
        a, b = part[..., :R // 2], part[..., R // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = part[..., 0::2], part[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _split_qkv(c: dict, qkv):
    N, Hq, Hkv, D = c["tokens"], c["heads"], c["kv_heads"], c["dim"]
    return (t.view(N, -1, D) for t in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=1))


def _rotary_plain(s: dict):
    c = s["case"]
    q, k, v = _split_qkv(c, s["qkv"])
    angle = s["pos"].double()[:, None] * s["freq"]  # far positions: 64 bits
    cos, sin = (f(angle).float() * s["factor"] for f in (torch.cos, torch.sin))
    s["out"].copy_(_rotate(q.float(), cos, sin, c["layout"]))
    page, at = s["slots"] // c["page"], s["slots"] % c["page"]
    s["k"][page, :, at] = _rotate(k.float(), cos, sin, c["layout"]).to(s["k"].dtype)
    s["v"][page, :, at] = v
    return s["out"], s["k"], s["v"]


def _verify_plain(s: dict):
    """All sequences together, a node after the other (a node is tested where
    its parent is the last accepted one), in 64 bits: values next to a border."""
    c = s["case"]
    B, T, V = c["batch"], c["nodes"], c["vocab"]
    rows = torch.arange(B, device="cuda")
    start, count = s["node_off"][:-1].long(), s["node_off"].diff().long()
    cur, tests, n_acc = (torch.zeros(B, dtype=torch.int64, device="cuda") for _ in range(3))
    none_left = torch.zeros(B, dtype=torch.bool, device="cuda")
    r, d = s["p"][start].double(), s["q"][start].double()
    W, Z = (torch.ones(B, dtype=torch.float64, device="cuda") for _ in range(2))
    path = torch.full((B, T), -1, dtype=torch.int64, device="cuda")
    toks = torch.full((B, T), -1, dtype=torch.int64, device="cuda")
    path[:, 0] = 0
    for i in range(1, T):
        at = torch.where(i < count, start + i, start)
        x = s["tokens"][at].long()
        test = (i < count) & (s["parents"][at] == cur) & ~none_left
        ratio = (r[rows, x] / W) / (d[rows, x] / Z)
        accept = test & ~(s["u"][rows, tests] >= torch.where(ratio < 1.0, ratio, 1.0))
        reject = test & ~accept
        tests += test
        toks[rows, n_acc] = torch.where(accept, x, toks[rows, n_acc])
        n_acc += accept
        path[rows, n_acc] = torch.where(accept, i, path[rows, n_acc])
        cur = torch.where(accept, i, cur)
        left = (r / W[:, None] - d / Z[:, None]).clamp_min(0.0)
        total = left.sum(1)
        none_left |= reject & (total == 0)
        left = torch.where((total == 0)[:, None], s["p"][start + cur].double(), left)
        r = torch.where(accept[:, None], s["p"][at].double(), torch.where(reject[:, None], left, r))
        W = torch.where(accept, 1.0, torch.where(reject, total, W))
        if not c["replacement"]:
            d[rows, x] = torch.where(reject, 0.0, d[rows, x])
        d = torch.where(accept[:, None], s["q"][at].double(), d)
        Z = torch.where(accept, 1.0, Z if c["replacement"] else torch.where(reject, d.sum(1), Z))
    sums = r.cumsum(1)
    toks[rows, n_acc] = (sums <= s["u"][rows, tests][:, None] * sums[:, -1:]).sum(1).clamp_max(V - 1)
    return tuple(t.to(torch.int32) for t in (toks, path, n_acc, tests + 1))


def _copy_plain(s: dict):
    for pool in (s["k"], s["v"]):
        pool[:, s["dst"].long()] = pool[:, s["src"].long()]
    return s["k"], s["v"]


def _keep_plain(s: dict):
    c = s["case"]
    j = torch.arange(c["nodes"], device="cuda")
    moved = j <= s["n"][:, None]
    lens, table = s["lens"].long()[:, None], s["table"].long()
    src, dst = lens + torch.where(moved, s["path"].long(), j), lens + j
    for pool in (s["k"], s["v"]):
        rows = pool[:, table.gather(1, src // c["page"]), :, src % c["page"]]
        pool[:, table.gather(1, dst // c["page"]), :, dst % c["page"]] = rows
    return s["k"], s["v"]


_PLAIN = {"attend": _attend_plain, "rotary": _rotary_plain, "verify": _verify_plain, "copy": _copy_plain,
          "keep": _keep_plain}


def run(s: dict):
    c = s["case"]
    if not own:
        return _PLAIN[c["kind"]](s)
    from pagellm_amd import cache, tree

    if c["kind"] == "attend":
        return tree.tree_attention(s["q"], s["k"], s["v"], s["table"], s["lens"], s["node_off"], s["visible"],
                                   max_nodes=c["nodes"], max_len=c["length"] + c["nodes"], out=s["out"])
    if c["kind"] == "rotary":
        q, k, v = _split_qkv(c, s["qkv"])
        cache.rotary_append(q, k, v, s["pos"], s["slots"], s["k"], s["v"], s["rotary"], q_out=s["out"])
        return s["out"], s["k"], s["v"]
    if c["kind"] == "verify":
        return tuple(tree.verify_tree(s["p"], s["q"], s["tokens"], s["parents"], s["node_off"], s["u"],
                                      max_nodes=c["nodes"], replacement=c["replacement"]))
    if c["kind"] == "copy":
        cache.copy_pages(s["k"], s["v"], s["src"], s["dst"])
    else:
        cache.keep_nodes(s["k"], s["v"], s["table"], s["lens"], s["path"], s["n"])
    return s["k"], s["v"]


def work(case: dict) -> dict:
    c = case
    e = _BYTES[c["dtype"]]
    if c["kind"] == "attend":  # trees and contexts are three quarters of their largest on average
        B, T, L = c["batch"], 0.75 * c["nodes"] if c["nodes"] > 1 else 1, 0.75 * c["length"]
        keys = L + T
        return {"bytes": int(B * (2 * keys * c["kv_heads"] + 2 * T * c["heads"]) * c["dim"] * e),
                "flops": int(4 * B * T * c["heads"] * c["dim"] * keys)}
    if c["kind"] == "rotary":
        n = c["tokens"] * (c["heads"] + 2 * c["kv_heads"]) * c["dim"]
        return {"bytes": 2 * n * e + 16 * c["tokens"], "flops": 3 * n}
    if c["kind"] == "verify":  # the rows in which the last token is drawn, and each test's two values
        return {"bytes": c["batch"] * (2 * c["vocab"] * e + 20 * c["nodes"]), "flops": 4 * c["batch"] * c["vocab"]}
    page = 2 * c["layers"] * c["kv_heads"] * c["dim"] * e  # a token's keys and values
    if c["kind"] == "copy":
        return {"bytes": 2 * c["pairs"] * c["page"] * page, "flops": 0}
    return {"bytes": max(1, c["batch"] * min(8, c["nodes"]) // 3) * 2 * page, "flops": 0}


# ------------------------------------------------- the same in plain float64


def _attend_exact(c: dict, d: dict):
    T, Hq, Hkv, D, ps = c["nodes"], c["heads"], c["kv_heads"], c["dim"], c["page"]
    out = torch.empty((d["q"].shape[0], Hq, D), dtype=torch.float64, device="cuda")
    off, lens = d["node_off"].tolist(), d["lens"].tolist()
    for b in range(c["batch"]):
        n = off[b + 1] - off[b]
        L = lens[b] + n
        pages = d["table"][b, : -(-L // ps)].long()
        k, v = (d[x][pages].transpose(0, 1).reshape(Hkv, -1, D)[:, :L].double() for x in ("k", "v"))
        sees = torch.ones((n, L), dtype=torch.bool, device="cuda")
        for i in range(n):
            if d["visible"] is None:
                sees[i, lens[b] + i + 1:] = False
            else:
                bits = int(d["visible"][off[b] + i])
                sees[i, lens[b]:] = torch.tensor([bits >> m & 1 == 1 for m in range(n)], device="cuda")
        for h in range(Hkv):
            g = Hq // Hkv
            q = d["q"][off[b]:off[b + 1], h * g:(h + 1) * g].double()
            x = (q.reshape(n * g, D) @ k[h].T.contiguous()).view(n, g, L) / math.sqrt(D)
            w = torch.softmax(x.masked_fill(~sees[:, None], -math.inf), -1)
            out[off[b]:off[b + 1], h * g:(h + 1) * g] = (w.view(n * g, L) @ v[h]).view(n, g, D)
    return out


def _rotary_exact(c: dict, d: dict):
    turn = torch.polar(torch.full_like(d["freq"], d["factor"]).expand(c["tokens"], -1),
                       d["pos"].double()[:, None] * d["freq"])[:, None]
    R, outs = c["part"], []
    q, k, v = (t.double() for t in _split_qkv(c, d["qkv"]))
    for x in (q, k):
        y = x.clone()
        if c["layout"] == "half":
            z = torch.complex(x[..., :R // 2], x[..., R // 2:R]) * turn
            y[..., :R // 2], y[..., R // 2:R] = z.real, z.imag
        else:
            z = torch.view_as_complex(x[..., :R].reshape(*x.shape[:2], R // 2, 2)) * turn
            y[..., :R] = torch.view_as_real(z).flatten(-2)
        outs.append(y)
    pools = []
    for pool, new in ((d["k"], outs[1]), (d["v"], v)):
        flat = pool.double().transpose(1, 2).reshape(-1, c["kv_heads"], c["dim"])
        flat[d["slots"]] = new
        pools.append(flat.view(-1, c["page"], c["kv_heads"], c["dim"]).transpose(1, 2).contiguous())
    return outs[0], pools[0], pools[1]


def _copy_exact(c: dict, d: dict):
    k, v = d["k"].double(), d["v"].double()
    for a, b in zip(d["src"].tolist(), d["dst"].tolist()):
        k[:, b], v[:, b] = d["k"][:, a].double(), d["v"][:, a].double()
    return k, v


def _keep_exact(c: dict, d: dict):
    k, v, ps = d["k"].double(), d["v"].double(), c["page"]
    table, lens, path, n = (d[x].tolist() for x in ("table", "lens", "path", "n"))
    for b in range(c["batch"]):
        for j in range(1, n[b] + 1):
            a, z = lens[b] + path[b][j], lens[b] + j
            for new, old in ((k, d["k"]), (v, d["v"])):
                new[:, table[b][z // ps], :, z % ps] = old[:, table[b][a // ps], :, a % ps].double()
    return k, v


def exact(case: dict, seed: int):
    """What run() returns, in plain float64 (None for whole numbers)."""
    if case["kind"] == "verify":
        return None
    d = _INPUTS[case["kind"]](case, seed)
    return {"attend": _attend_exact, "rotary": _rotary_exact, "copy": _copy_exact, "keep": _keep_exact}[case["kind"]](case, d)
