"""What the operators for drafted tokens and for pages of the cache are timed on.

A request whose next tokens were drafted as a tree runs them in one step: the drafted tokens' keys and values stand in
the cache behind the request's own, a mask says which of them each sees (``attention``; the mask comes from the
tokens' parents, ``tree``), the tokens the model itself would have chosen are followed down the tree and the cache keeps
the accepted ones alone, side by side (``accept``).  Pages of the cache are copied when a request is forked or the
pool is put together (``copy``).

Sizes: heads and layers of the benchmark's Qwen3 configurations (8B: 32 query heads, 14B: 40, 32B: 64; 8 KV heads of 128,
36 layers), pages of 16 tokens, contexts up to 32,768 tokens, and smaller heads, other pages and float32 beside them.
"""
import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed():
    return [
        # one user, a chain of five drafted tokens: the smallest call, all latency
        {"name": "attention_chain_1x5", "kind": "attention", "batch": 1, "nodes_lo": 5, "nodes": 5, "chain": True, "ctx_lo": 600,
         "ctx": 600, "nq": 32, "nkv": 8, "hd": 128, "page": 16, "window": 0, "dtype": "bf16", "mix": 1},
        # one user behind a long document, a tree of 24: few rows, many keys
        {"name": "attention_1x24_behind_16k", "kind": "attention", "batch": 1, "nodes_lo": 24, "nodes": 24, "chain": False,
         "ctx_lo": 16000, "ctx": 16000, "nq": 32, "nkv": 8, "hd": 128, "page": 16, "window": 0, "dtype": "bf16", "mix": 2},
        # a serving batch of 8B sizes, trees of up to 32 tokens behind contexts of unlike length
        {"name": "attention_8x32_behind_2k", "kind": "attention", "batch": 8, "nodes_lo": 20, "nodes": 32, "chain": False,
         "ctx_lo": 1000, "ctx": 3000, "nq": 32, "nkv": 8, "hd": 128, "page": 16, "window": 0, "dtype": "bf16", "mix": 3},
        # the largest: 14B heads, trees of 64 behind contexts of up to 32,768 tokens
        {"name": "attention_8x64_behind_32k", "kind": "attention", "batch": 8, "nodes_lo": 64, "nodes": 64, "chain": False,
         "ctx_lo": 16000, "ctx": 32768, "nq": 40, "nkv": 8, "hd": 128, "page": 16, "window": 0, "dtype": "bf16", "mix": 4},
        # heads of 64 under a sliding window, pages of an odd size, ragged trees
        {"name": "attention_window_6x40", "kind": "attention", "batch": 6, "nodes_lo": 3, "nodes": 40, "chain": False,
         "ctx_lo": 30, "ctx": 2500, "nq": 16, "nkv": 4, "hd": 64, "page": 20, "window": 1000, "dtype": "bf16", "mix": 5},
        # the true 32-bit path
        {"name": "attention_float32_3x12", "kind": "attention", "batch": 3, "nodes_lo": 9, "nodes": 12, "chain": False,
         "ctx_lo": 500, "ctx": 1500, "nq": 16, "nkv": 8, "hd": 64, "page": 16, "window": 0, "dtype": "f32", "mix": 6},
        # the mask of a small batch's trees, and of many wide ones
        {"name": "tree_8x32", "kind": "tree", "batch": 8, "nodes_lo": 20, "nodes": 32, "chain": False, "ctx": 2000, "window": 0,
         "mix": 7},
        {"name": "tree_64x256", "kind": "tree", "batch": 64, "nodes_lo": 200, "nodes": 256, "chain": False, "ctx": 8000,
         "window": 0, "mix": 8},
        # one user's accepted tokens kept in every layer, and a batch's
        {"name": "accept_1x8", "kind": "accept", "batch": 1, "nodes": 8, "accepted": 3, "layers": 36, "nkv": 8, "hd": 128,
         "page": 16, "ctx": 500, "dtype": "bf16", "mix": 9},
        {"name": "accept_32x64", "kind": "accept", "batch": 32, "nodes": 64, "accepted": 7, "layers": 36, "nkv": 8, "hd": 128,
         "page": 16, "ctx": 100, "dtype": "bf16", "mix": 10},
        # a fork of one request: its last page; and many pages at once, as when a pool's live pages are put together
        {"name": "copy_1", "kind": "copy", "pages": 1, "layers": 36, "nkv": 8, "hd": 128, "page": 16, "dtype": "bf16", "mix": 11},
        {"name": "copy_256", "kind": "copy", "pages": 256, "layers": 36, "nkv": 8, "hd": 128, "page": 16, "dtype": "bf16",
         "mix": 12},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention", "tree", "accept", "copy"])
    mix = rng.randint(0, 10 ** 6)
    if kind == "attention":
        dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
        nodes, nkv, g = _spread(rng, 1, 64), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 8])
        batch = _spread(rng, 1, 32)
        hd = rng.choice([64, 128, 128, 128, 16 * rng.randint(1, 16)])
        # rows x keys, and keys alone, of the batch stay below those of the largest listed case
        most = min(32768 if dtype == "bf16" else 4096, 8 * 64 * 40 * 24000 * 128 // (batch * nodes * nkv * g * hd),
                   8 * 24000 * 8 * 128 // (batch * nkv * hd))
        ctx = _spread(rng, 1, max(1, most))
        return {"kind": kind, "batch": batch, "nodes_lo": rng.randint(1, nodes), "nodes": nodes, "chain": rng.random() < 0.25,
                "ctx_lo": rng.randint(0, ctx), "ctx": ctx, "nq": nkv * g, "nkv": nkv,
                "hd": hd, "page": rng.choice([8, 16, 16, 32, 64, rng.randint(3, 48)]),
                "window": rng.choice([0, 0, 0, _spread(rng, 2, 4096)]), "dtype": dtype, "mix": mix}
    if kind == "tree":
        nodes = _spread(rng, 1, 256)
        return {"kind": kind, "batch": _spread(rng, 1, 64), "nodes_lo": rng.randint(1, nodes), "nodes": nodes,
                "chain": rng.random() < 0.25, "ctx": _spread(rng, 1, 30000), "window": rng.choice([0, 0, _spread(rng, 2, 1000)]), "mix": mix}
    dtype = rng.choice(["bf16", "bf16", "f32"])
    layers, nkv, hd, page = rng.randint(1, 36), rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 8 * rng.randint(2, 32)]), rng.choice([8, 16, 32])
    if kind == "accept":
        accepted = rng.randint(1, 8)
        return {"kind": kind, "batch": _spread(rng, 1, 32), "nodes": rng.randint(2 * accepted, 64), "accepted": accepted, "layers": layers,
                "nkv": nkv, "hd": hd, "page": page, "ctx": _spread(rng, 1, 100), "dtype": dtype, "mix": mix}
    size = layers * nkv * hd * page * (2 if dtype == "bf16" else 4)
    pages = _spread(rng, 1, max(1, min(512, 256 * 36 * 8 * 128 * 16 * 2 // size)))
    return {"kind": kind, "pages": pages, "layers": layers, "nkv": nkv, "hd": hd, "page": page, "dtype": dtype, "mix": mix}


def _lengths(case):
    """(tokens, committed tokens) of every request; the case's own, whatever the inputs' seed."""
    rng = random.Random(case["mix"])
    lo = case.get("nodes_lo", case["nodes"])
    nodes = [case["nodes"]] + [rng.randint(lo, case["nodes"]) for _ in range(case["batch"] - 1)]
    ctx = [case["ctx"]] + [rng.randint(case.get("ctx_lo", 0), case["ctx"]) for _ in range(case["batch"] - 1)]
    return nodes, ctx


def _accepted(case):
    """Tokens kept of every request, the first of each among them."""
    return [1 + (case["accepted"] - 1 + 3 * e) % case["accepted"] for e in range(case["batch"])]


def _parents(case, nodes, r):
    """Parents of every request's tokens within the request, -1 for the first: chains, or trees as a drafter's beam grows
    them, a token's parent among the few before it."""
    if case.get("chain"):
        return [np.arange(-1, q - 1) for q in nodes]
    trees = []
    for q in nodes:
        i = np.arange(q)
        back = 1 + (r.rand(q) * (1 + i / 3)).astype(np.int64)
        p = np.maximum(i - back, 0)
        p[0] = -1
        trees.append(p)
    return trees


def _ints(a):
    return torch.from_numpy(np.ascontiguousarray(a)).to(torch.int32).to(DEV)


def _cache(case, kv, gen, slabs=()):
    """(pools, block table) of requests that hold ``kv`` tokens each, on pages in no order."""
    ps = case["page"]
    need = [-(-k // ps) for k in kv]
    pages = sum(need) + 3
    order = np.random.RandomState(case["mix"]).permutation(pages)
    table = np.zeros((len(kv), max(need)), dtype=np.int32)
    at = 0
    for e, k in enumerate(need):
        table[e, :k] = order[at:at + k]
        at += k
    pools = [torch.randn(tuple(slabs) + (pages, case["nkv"], ps, case["hd"]), generator=gen, device=DEV,
                         dtype=DT[case["dtype"]]) for _ in range(1 if slabs else 2)]
    return pools, _ints(table)


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    r = np.random.RandomState(seed % (2 ** 31))
    s = dict(case)
    if case["kind"] == "copy":
        n = case["pages"]
        order = np.random.RandomState(case["mix"]).permutation(2 * n + 6)
        s["src"], s["dst"] = order[:n].tolist(), order[n:2 * n].tolist()
        s["src_dev"], s["dst_dev"] = _ints(order[:n]).long(), _ints(order[n:2 * n]).long()
        s["pool"] = torch.randn((case["layers"], 2, 2 * n + 6, case["nkv"], case["page"], case["hd"]), generator=gen, device=DEV,
                                dtype=DT[case["dtype"]])
        return s
    nodes, ctx = _lengths(case)
    if case["kind"] == "tree":
        ctx = [c + int(r.randint(0, 1000)) for c in ctx]       # a chain's own mask is always the same
    kv = [c + q for c, q in zip(ctx, nodes)]
    T, n, Q = sum(nodes), case["batch"], max(nodes)
    cu = np.concatenate([[0], np.cumsum(nodes)])
    s["cu_q"], s["kv_lens"], s["max_q"] = _ints(cu), _ints(np.array(kv)), Q
    words = -(-Q // 32)
    if case["kind"] in ("attention", "tree"):
        trees = _parents(case, nodes, r)
        s["parents"] = _ints(np.concatenate(trees))
        s["positions"] = torch.zeros(T, dtype=torch.int32, device=DEV)
        s["mask"] = torch.zeros((T, words), dtype=torch.int32, device=DEV)
    if case["kind"] == "attention":
        # the mask stands from here on: a step makes it once for all of its layers
        s["positions"], s["mask"] = _plain_tree(s)
        (s["k"], s["v"]), s["table"] = _cache(case, kv, gen)
        s["q"] = torch.randn((T, case["nq"] * case["hd"]), generator=gen, device=DEV, dtype=DT[case["dtype"]])
        s["out"] = torch.empty_like(s["q"])
    if case["kind"] == "accept":
        # the path that the model's own tokens take; its places lie behind those it is moved to
        kept = _accepted(case)
        tokens, parents, targets = [], [], []
        for e, q in enumerate(nodes):
            a = kept[e]
            path = np.concatenate([[0], np.sort(r.choice(np.arange(a, q), size=a - 1, replace=False))]).astype(np.int64)
            p = _parents(case, [q], r)[0]
            p[path[1:]] = path[:-1]
            tok = r.permutation(30000)[:q]                    # no two alike: only the path's own child follows
            want = 30000 + r.randint(0, 1000, size=q)
            want[path[:-1]] = tok[path[1:]]
            tokens.append(tok), parents.append(p), targets.append(want)
        s["tokens"], s["parents"], s["targets"] = (_ints(np.concatenate(x)) for x in (tokens, parents, targets))
        s["path"] = torch.zeros((n, case["accepted"] + 1), dtype=torch.int32, device=DEV)
        s["count"], s["next"] = torch.zeros(n, dtype=torch.int32, device=DEV), torch.zeros(n, dtype=torch.int32, device=DEV)
        (s["pool"],), s["table"] = _cache(case, kv, gen, (case["layers"], 2))
    return s


def run(s):
    if own:
        from safetyraise_lmengine_b200.kernels import ops
        if s["kind"] == "attention":
            ops.tree_attention(s["q"], s["k"], s["v"], s["out"], s["table"], s["cu_q"], s["kv_lens"], s["mask"], s["nq"], s["nkv"],
                               s["hd"], s["page"], 1.0 / math.sqrt(s["hd"]), s["max_q"], positions=s["positions"],
                               window=s["window"])
            return s["out"]
        if s["kind"] == "tree":
            ops.draft_tree(s["parents"], s["cu_q"], s["kv_lens"], s["positions"], s["mask"], window=s["window"])
            return [s["positions"], s["mask"]]
        if s["kind"] == "accept":
            ops.accept_drafts(s["tokens"], s["parents"], s["targets"], s["cu_q"], s["path"], s["count"], s["next"])
            ops.keep_drafts(s["pool"], s["table"], s["cu_q"], s["kv_lens"], s["path"], s["count"])
            return [s["path"], s["count"], s["next"], s["pool"]]
        ops.copy_pages(s["pool"], s["src"], s["dst"])
        return s["pool"]
    if s["kind"] == "attention":
        return _plain_attention(s)
    if s["kind"] == "tree":
        return list(_plain_tree(s))
    if s["kind"] == "accept":
        return _plain_accept(s)
    s["pool"][:, :, s["dst_dev"]] = s["pool"][:, :, s["src_dev"]]
    return s["pool"]


def _padded(s, x, fill):
    """A tensor of one value a token as [requests, most tokens of one], and which of its places are tokens."""
    at = s["cu_q"][:-1, None].long() + torch.arange(s["max_q"], device=DEV)
    real = at < s["cu_q"][1:, None]
    return torch.where(real, x[at.clamp(max=x.shape[0] - 1)], fill), real


def _tokens(s, real, x):
    """The rows of a padded tensor that are tokens, in the batch's order (their number is the tokens': no wait for it)."""
    lens = s["cu_q"].long().diff()
    e = torch.repeat_interleave(torch.arange(lens.shape[0], device=DEV), lens, output_size=s["parents"].shape[0])
    return x[e, torch.arange(s["parents"].shape[0], device=DEV) - s["cu_q"].long()[e]]


def _plain_tree(s):
    """Positions and mask bits: the tokens from which a token descends are those that powers of (identity + parents) reach."""
    Q = s["max_q"]
    parents, real = _padded(s, s["parents"], -1)
    j = torch.arange(Q, device=DEV)
    reach = ((j == j[:, None]) | (parents[:, :, None] == j)).float()
    for _ in range(max(1, (Q - 1).bit_length())):
        reach = (reach @ reach > 0).float()
    depth = reach.sum(-1) - 1
    if s["window"]:
        reach = reach * (depth[:, :, None] - depth[:, None, :] < s["window"])
    q_lens = s["cu_q"].diff()
    positions = _tokens(s, real, (s["kv_lens"] - q_lens)[:, None] + depth.to(torch.int32))
    words = s["mask"].shape[1]
    bits = torch.zeros(reach.shape[:2] + (words * 32,), dtype=torch.int64, device=DEV)
    bits[:, :, :Q] = reach.long()
    packed = (bits.view(*reach.shape[:2], words, 32) << torch.arange(32, device=DEV)).sum(-1)
    packed = (packed ^ 0x80000000) - 0x80000000                    # 32 bits as a signed number
    return positions, _tokens(s, real, packed.to(torch.int32))


def _plain_attention(s):
    n, Q, g, hd = s["kv_lens"].shape[0], s["max_q"], s["nq"] // s["nkv"], s["hd"]
    # keys and values in order, [requests, KV heads, places, head size]
    k, v = (c[s["table"].long()].transpose(1, 2).flatten(2, 3).float() for c in (s["k"], s["v"]))
    places = k.shape[2]
    at = (s["cu_q"][:-1, None].long() + torch.arange(Q, device=DEV)).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float().view(-1, s["nkv"], g, hd)[at].permute(0, 2, 3, 1, 4).reshape(n, s["nkv"], g * Q, hd)
    scores = (q @ k.transpose(2, 3)).view(n, s["nkv"], g, Q, places) / math.sqrt(hd)
    j = torch.arange(places, device=DEV)
    start = (s["kv_lens"] - s["cu_q"].diff())[:, None, None]
    node = (j - start).clamp(0, 32 * s["mask"].shape[1] - 1).expand(n, Q, places)
    bit = (s["mask"][at].long().gather(2, node // 32) >> (node % 32)) & 1
    position = s["positions"][at][:, :, None]
    committed = (j < start) & ((position - j < s["window"]) if s["window"] else True)
    seen = torch.where(j < start, committed, (j < s["kv_lens"][:, None, None]) & (bit == 1))
    scores = scores.masked_fill(~seen[:, None, None], -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = (p / p.sum(-1, keepdim=True)).view(n, s["nkv"], g * Q, places)
    # a place behind a request's last key is on no page of its own
    v = torch.where((j < start[:, 0] + s["cu_q"].diff()[:, None])[:, None, :, None], v, 0.0)
    o = (p @ v).view(n, s["nkv"], g, Q, hd).permute(0, 3, 1, 2, 4).reshape(n, Q, -1)
    return _tokens(s, None, o).to(s["q"].dtype)


def _plain_accept(s):
    n, cap = s["path"].shape
    tokens, real = _padded(s, s["tokens"], -1)
    parents, targets = _padded(s, s["parents"], -2)[0], _padded(s, s["targets"], -1)[0]
    e = torch.arange(n, device=DEV)
    path, live = s["path"], torch.ones(n, dtype=torch.bool, device=DEV)
    cur = torch.zeros(n, dtype=torch.long, device=DEV)
    path[:, 0] = 0
    for i in range(1, cap):
        hit = (parents == cur[:, None]) & (tokens == targets[e, cur][:, None]) & real & live[:, None]
        live = hit.any(1)
        cur = torch.where(live, hit.int().argmax(1), cur)
        path[:, i] = torch.where(live, cur, -1)
    s["count"][:] = (path >= 0).sum(1)
    s["next"][:] = targets[e, cur]
    # the kept tokens' rows; what is not kept stays where it is
    i = torch.arange(cap, device=DEV)
    start = (s["kv_lens"] - s["cu_q"].diff())[:, None]
    last = s["kv_lens"][:, None] - 1
    to = torch.minimum(start + i, last).long()
    frm = torch.where(path >= 0, (start + path).long(), to)
    ps, row = s["page"], e[:, None]
    s["pool"][:, :, s["table"].long()[row, to // ps], :, to % ps] = s["pool"][:, :, s["table"].long()[row, frm // ps], :, frm % ps]
    return [path, s["count"], s["next"], s["pool"]]


def exact(case, seed):
    """Attention from its definition, request by request in 64 bits.  The other operators move data or count."""
    if case["kind"] != "attention":
        return None
    s = prepare(case, seed)
    cu, kv, table = s["cu_q"].tolist(), s["kv_lens"].tolist(), s["table"].long()
    parents = s["parents"].tolist()
    g, hd, nkv = case["nq"] // case["nkv"], case["hd"], case["nkv"]
    out = torch.zeros((cu[-1], case["nq"], hd), dtype=torch.float64, device=DEV)
    for e in range(case["batch"]):
        q_len, start = cu[e + 1] - cu[e], kv[e] - (cu[e + 1] - cu[e])
        up = parents[cu[e]:cu[e + 1]]
        seen, depths = np.zeros((q_len, kv[e]), dtype=bool), []
        for i in range(q_len):
            line = [i]
            while up[line[-1]] >= 0:
                line.append(up[line[-1]])
            depths.append(len(line) - 1)
            first = max(0, start + depths[i] - case["window"] + 1) if case["window"] else 0
            seen[i, first:start] = True
            for j in line:
                seen[i, start + j] = not case["window"] or depths[i] - depths[j] < case["window"]
        seen = torch.from_numpy(seen).to(DEV)
        pages = table[e, :-(-kv[e] // case["page"])]
        for h in range(nkv):
            kh = s["k"][pages, h].reshape(-1, hd)[:kv[e]].double()
            vh = s["v"][pages, h].reshape(-1, hd)[:kv[e]].double()
            for i in range(h * g, (h + 1) * g):
                qh = s["q"][cu[e]:cu[e + 1], i * hd:(i + 1) * hd].double()
                w = torch.softmax((qh @ kh.T / math.sqrt(hd)).masked_fill(~seen, -math.inf), dim=1)
                out[cu[e]:cu[e + 1], i] = w @ vh
    return out.view(cu[-1], -1)


def work(case):
    size = 2 if case.get("dtype") == "bf16" else 4
    if case["kind"] == "copy":
        return {"bytes": 2 * case["pages"] * case["layers"] * 2 * case["nkv"] * case["page"] * case["hd"] * size, "flops": 0}
    nodes, ctx = _lengths(case)
    T, words = sum(nodes), -(-max(nodes) // 32)
    if case["kind"] == "tree":
        return {"bytes": 4 * (2 * T + T * words + 2 * case["batch"] + 1), "flops": 0}
    if case["kind"] == "accept":
        moved = sum(a - 1 for a in _accepted(case))
        return {"bytes": 2 * moved * case["layers"] * 2 * case["nkv"] * case["hd"] * size
                + 4 * (3 * T + case["batch"] * (case["accepted"] + 5)), "flops": 0}
    w, row = case["window"], case["hd"] * size
    # committed keys: those the window leaves the first token, and the rows that see each
    keys = [min(c, w - 1) if w else c for c in ctx]
    pairs = sum(q * k for q, k in zip(nodes, keys)) + T
    return {"bytes": 2 * row * case["nkv"] * (sum(keys) + T) + 2 * row * case["nq"] * T + 4 * T * words
            + 4 * sum(-(-k // case["page"]) for k in keys),
            "flops": 4 * case["hd"] * case["nq"] * pairs}
