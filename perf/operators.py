"""Ragged prompts, drafted trees and token probabilities as cases that can be timed and checked.

Four operators that serve a batch of sequences of different lengths:

* ``packed_attention``: causal GQA attention of the packed prompt rows of many sequences
  (fresh prompts, later chunks of long prompts, single tokens among them) over the cache;
* ``tree_attention``: attention of a tree of drafted tokens over each sequence's cache;
* ``tree_commit``: the accepted path of such a tree, and its K/V rows moved to the front;
* ``token_logprobs``: log probabilities of given tokens, entropy and top alternatives.

With ``own`` false ``run`` computes them from elementary torch operations in float32,
rounded once at the end; with ``own`` true it makes the package's calls.  ``exact``
computes the same from the definitions in float64.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
BF16 = torch.bfloat16
D = 128            # head dimension
VOCAB = 151936
TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # three chat turns arriving together: the smallest packed call, latency
        {"name": "packed_3_short", "kind": "packed", "hq": 16, "hkv": 8, "cap": 320, "n": 3, "lo": 1, "hi": 43,
         "p_lo": 0, "p_hi": 0, "singles": 0},
        # a serving batch of fresh prompts of different lengths
        {"name": "packed_16", "kind": "packed", "hq": 16, "hkv": 8, "cap": 1088, "n": 16, "lo": 37, "hi": 1021,
         "p_lo": 0, "p_hi": 0, "singles": 0},
        # a mixed step: chunks of two long prompts among sequences that decode one token each
        {"name": "packed_chunks_24_singles", "kind": "packed", "hq": 32, "hkv": 8, "cap": 4800, "n": 2, "lo": 509,
         "hi": 701, "p_lo": 2005, "p_hi": 3990, "singles": 24},
        # one long document
        {"name": "packed_8001", "kind": "packed", "hq": 32, "hkv": 8, "cap": 8192, "n": 1, "lo": 8001, "hi": 8001,
         "p_lo": 0, "p_hi": 0, "singles": 0},
        # single stream with a small drafted tree: latency
        {"name": "tree_1x8", "kind": "tree", "hq": 16, "hkv": 8, "cap": 1088, "b": 1, "nodes": 8, "lo": 700, "hi": 700},
        # a serving batch, each sequence with its tree
        {"name": "tree_16x26", "kind": "tree", "hq": 16, "hkv": 8, "cap": 4096, "b": 16, "nodes": 26, "lo": 901,
         "hi": 4001},
        # wide trees over long contexts, four q heads a kv head
        {"name": "tree_8x64_long", "kind": "tree", "hq": 32, "hkv": 8, "cap": 32768, "b": 8, "nodes": 64, "lo": 15007,
         "hi": 32003},
        # the accepted path of one sequence in the cache of 28 layers: latency
        {"name": "commit_1x8", "kind": "commit", "layers": 28, "hkv": 8, "cap": 320, "b": 1, "nodes": 8},
        # the same for a batch
        {"name": "commit_32x26", "kind": "commit", "layers": 28, "hkv": 8, "cap": 320, "b": 32, "nodes": 26},
        # the alternatives of one decoded token
        {"name": "logprobs_1", "kind": "logprobs", "m": 1, "v": VOCAB, "type": "fp32", "k": 5},
        # every node of a batch's trees, half-precision logits
        {"name": "logprobs_416_bf16", "kind": "logprobs", "m": 416, "v": VOCAB, "type": "bf16", "k": 8},
        # scoring a prompt: every row, with the twenty best alternatives
        {"name": "logprobs_2043", "kind": "logprobs", "m": 2043, "v": VOCAB, "type": "fp32", "k": 20},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges."""
    kind = rng.choice(["packed", "packed", "packed", "tree", "tree", "commit", "logprobs", "logprobs"])
    hkv, g = rng.choice([(8, 2), (8, 4), (8, 1), (4, 8), (2, 7), (8, 3)])
    if kind == "packed":
        n = rng.choice([1, 1, 2, 3, 7, 16, 32])
        singles = rng.choice([0, 0, rng.randrange(1, 33)])
        hi = _log(rng, 2, 3900 if n < 3 else 900 if n < 8 else 500)
        p_hi = rng.choice([0, _log(rng, 1, 2000 if n < 3 else 4000 if n < 8 else 1000)])
        return {"kind": kind, "hq": hkv * g, "hkv": hkv, "cap": hi + p_hi + rng.randrange(0, 200), "n": n,
                "lo": rng.randrange(1, hi + 1), "hi": hi, "p_lo": rng.randrange(0, p_hi + 1), "p_hi": p_hi,
                "singles": singles}
    if kind == "tree":
        b = _log(rng, 1, 32)
        hi = _log(rng, 1, min(32000, 160000 // b))
        nodes = _log(rng, 1, 64)
        return {"kind": kind, "hq": hkv * g, "hkv": hkv, "cap": hi + nodes + rng.randrange(0, 700), "b": b,
                "nodes": nodes, "lo": rng.randrange(0, hi + 1), "hi": hi}
    if kind == "commit":
        nodes = _log(rng, 1, 64)
        return {"kind": kind, "layers": rng.randrange(1, 29), "hkv": hkv, "cap": nodes + rng.randrange(8, 220),
                "b": _log(rng, 1, 32), "nodes": nodes}
    m, v = _log(rng, 1, 2000), rng.choice([VOCAB, VOCAB, 4096, _log(rng, 1000, 150000)])
    return {"kind": kind, "m": m, "v": v, "type": rng.choice(["fp32", "fp32", "bf16", "fp16"]),
            "k": rng.randrange(0, 21)}


# ---- inputs, from the seed alone ----

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g).to(BF16)


def _sequences(case):
    """(rows, slots before them) of each packed sequence: rows spread over their logarithm
    from lo to hi, earlier slots evenly; then the sequences of one row."""
    n, lo, hi = case["n"], case["lo"], case["hi"]
    p_lo, p_hi, s = case["p_lo"], case["p_hi"], case["singles"]
    some = [(round(lo * (hi / lo) ** (i / max(n - 1, 1))) if n > 1 else hi,
             p_hi - (p_hi - p_lo) * i // max(n - 1, 1)) for i in range(n)]
    return some + [(1, p_lo + (p_hi - p_lo) * i // max(s - 1, 1)) for i in range(s)]


def _contexts(case):
    b, lo, hi = case["b"], case["lo"], case["hi"]
    return [hi - (hi - lo) * i // max(b - 1, 1) for i in range(b)]


def _parents(g, b, n):
    """Trees as a drafter grows them: each node hangs from one of the nodes before it,
    the likelier the nearer to the root; node 0 is the root."""
    i = torch.arange(n, device=DEV)
    u = torch.rand(b, n, device=DEV, generator=g)
    p = (u * u * i).long().clamp(max=max(n - 1, 0))
    p = torch.minimum(p, (i - 1).clamp(min=0))
    p[:, 0] = -1
    return p.to(torch.int32)


def _draft(g, b, n, parents):
    """Drafted tokens and the model's pick after every node: of a small set, so that
    paths of some nodes are accepted and siblings repeat a token now and then."""
    tokens = torch.randint(0, 6, (b, n), device=DEV, generator=g, dtype=torch.int32)
    picks = torch.randint(0, 6, (b, n), device=DEV, generator=g, dtype=torch.int32)
    hit = torch.rand(b, n, device=DEV, generator=g) < 0.7          # the drafter is mostly right
    at = parents.clamp(min=0).long()
    return torch.where(hit, picks.gather(1, at), tokens), picks


def prepare(case, seed):
    g, kind = _gen(seed), case["kind"]
    s = {"case": case}
    if kind == "packed":
        seqs = _sequences(case)
        random.Random(seed).shuffle(seqs)
        s["lens"], s["starts"] = [a for a, _ in seqs], [b for _, b in seqs]
        s["q"] = _normal(g, sum(s["lens"]), case["hq"], D)
        s["k_cache"], s["v_cache"] = (_normal(g, len(seqs), case["hkv"], case["cap"], D) for _ in range(2))
        if own:
            from torch2iron_amd import ops
            s["plan"] = ops.PackedPlan(s["lens"], case["hq"], case["hkv"], case["cap"], DEV, starts=s["starts"])
            s["workspace"] = ops.Workspace()
        else:   # where each packed row stands in the padded batch
            seq = torch.repeat_interleave(torch.arange(len(seqs)), torch.tensor(s["lens"]))
            first = torch.tensor([0] + s["lens"]).cumsum(0)[:-1]
            s["row_seq"] = seq.to(DEV)
            s["row_t"] = (torch.arange(len(seq)) - first[seq]).to(DEV)
            s["start"] = torch.tensor(s["starts"]).to(DEV)
    elif kind == "tree":
        b, n = case["b"], case["nodes"]
        ctx = torch.tensor(_contexts(case), dtype=torch.int32, device=DEV)
        s["ctx"] = ctx[torch.randperm(b, device=DEV, generator=g)].contiguous()
        s["parents"] = _parents(g, b, n)
        s["q"] = _normal(g, b, n, case["hq"], D)
        s["k_cache"], s["v_cache"] = (_normal(g, b, case["hkv"], case["cap"], D) for _ in range(2))
        if own:
            from torch2iron_amd import ops
            s["workspace"] = ops.Workspace()
    elif kind == "commit":
        b, n = case["b"], case["nodes"]
        s["parents"] = _parents(g, b, n)
        s["tokens"], s["picks"] = _draft(g, b, n, s["parents"])
        s["ctx"] = torch.randint(0, case["cap"] - n + 1, (b,), device=DEV, generator=g, dtype=torch.int32)
        shape = (case["layers"], b, case["hkv"], case["cap"], D)
        s["k_cache"], s["v_cache"] = (_normal(g, *shape) for _ in range(2))
    else:
        m, v = case["m"], case["v"]
        x = torch.randn(m, v, device=DEV, generator=g)
        x *= 2.0 + torch.rand(m, 1, device=DEV, generator=g)       # some rows surer than others
        s["logits"] = x.to(TYPES[case["type"]])
        s["tokens"] = torch.randint(0, v, (m,), device=DEV, generator=g, dtype=torch.int32)
        if own:
            from torch2iron_amd import ops
            s["workspace"] = ops.Workspace()
    return s


# ---- the operators ----

def _masked_attention(q, k, v, seen):
    """softmax(q k^T / sqrt(D)) v over the seen keys, float32: q [B, Hkv, R, D], k and v
    [B, Hkv, K, D], seen [B, 1, R, K]."""
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(D)
    x = x.masked_fill(~seen, -math.inf)
    w = torch.exp(x - x.amax(-1, keepdim=True))
    return torch.matmul(w, v) / w.sum(-1, keepdim=True)


def _ancestors(parents):
    """[B, N, N] whether node j is node i or above it."""
    n = parents.shape[1]
    i = torch.arange(n, device=DEV)
    up = (parents.long()[:, :, None] == i) | (i[:, None] == i)     # one step or none
    for _ in range(max(1, math.ceil(math.log2(max(n, 2))))):
        up = torch.matmul(up.float(), up.float()) > 0
    return up


def _packed(s):
    case = s["case"]
    hq, hkv = case["hq"], case["hkv"]
    b, t, keys = len(s["lens"]), max(s["lens"]), max(a + c for a, c in zip(s["lens"], s["starts"]))
    q = torch.zeros(b, t, hq, D, dtype=torch.float32, device=DEV)
    q[s["row_seq"], s["row_t"]] = s["q"].float()
    q = q.view(b, t, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, D)      # rows (head, t)
    pos = s["start"][:, None] + torch.arange(t, device=DEV)
    seen = torch.arange(keys, device=DEV) <= pos[:, :, None]                               # [B, T, K]
    seen = seen[:, None].expand(b, hq // hkv, t, keys).reshape(b, 1, -1, keys)
    o = _masked_attention(q, s["k_cache"][:, :, :keys].float(), s["v_cache"][:, :, :keys].float(), seen)
    o = o.view(b, hq, t, D).transpose(1, 2)[s["row_seq"], s["row_t"]]
    return o.reshape(-1, hq * D).to(BF16)


def _tree(s):
    case = s["case"]
    b, n, hq, hkv = case["b"], case["nodes"], case["hq"], case["hkv"]
    keys = case["hi"] + n
    slot = torch.arange(keys, device=DEV)
    ctx = s["ctx"].long()[:, None]
    node = slot - ctx                                                                      # [B, K]
    of_tree = (node >= 0) & (node < n)
    up = _ancestors(s["parents"]).gather(2, node.clamp(0, n - 1)[:, None].expand(b, n, keys))
    seen = (slot < ctx)[:, None] | (of_tree[:, None] & up)                                 # [B, N, K]
    g = hq // hkv
    q = s["q"].float().view(b, n, hkv, g, D).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, D)
    seen = seen[:, None].expand(b, g, n, keys).reshape(b, 1, -1, keys)
    o = _masked_attention(q, s["k_cache"][:, :, :keys].float(), s["v_cache"][:, :, :keys].float(), seen)
    return o.view(b, hq, n, D).transpose(1, 2).reshape(b * n, hq * D).to(BF16)


def _commit(s):
    tokens, picks, parents, ctx = s["tokens"], s["picks"], s["parents"].long(), s["ctx"].long()
    b, n = tokens.shape
    i = torch.arange(n, device=DEV)
    right = (parents >= 0) & (tokens == picks.gather(1, parents.clamp(min=0)))
    twin = (parents[:, :, None] == parents[:, None]) & right[:, None] & (i < i[:, None])   # an earlier right sibling
    right &= ~twin.any(-1)
    right[:, 0] = True
    wrong_above = _ancestors(s["parents"]) & ~right[:, None]
    # a node without a parent is above no path but node 0's
    taken = ~wrong_above.any(-1)
    counts = taken.sum(-1)
    path = torch.where(taken, i, n).sort(-1).values                                        # in order of the walk
    live = path < n
    dst = ctx[:, None] + i
    src = torch.where(live, ctx[:, None] + path, dst)
    rows = torch.arange(b, device=DEV)[:, None]
    for c in (s["k_cache"], s["v_cache"]):
        c[:, rows, :, dst] = c[:, rows, :, src]
    last = path.gather(1, counts[:, None] - 1)
    return {"path": torch.where(live, path, -1).to(torch.int32), "counts": counts.to(torch.int32),
            "next": picks.gather(1, last)[:, 0], "context": (ctx + counts).to(torch.int32),
            "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _logprobs(s):
    x, k = s["logits"].float(), s["case"]["k"]
    m = x.amax(-1, keepdim=True)
    e = torch.exp(x - m)
    z = e.sum(-1, keepdim=True)
    lse = m + torch.log(z)
    out = {"logprobs": x.gather(1, s["tokens"].long()[:, None])[:, 0] - lse[:, 0],
           "entropy": torch.log(z)[:, 0] - (e * (x - m)).sum(-1) / z[:, 0]}
    # best first, the lower index of equal values first: one whole number of both
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    key = order * (1 << 32) + ((1 << 32) - 1 - torch.arange(x.shape[1], device=DEV))
    ids = (1 << 32) - 1 - (key.topk(k, -1).values & ((1 << 32) - 1))
    return {**out, "top_logprobs": x.gather(1, ids) - lse, "top_ids": ids.to(torch.int32)}


def run(s):
    case, kind = s["case"], s["case"]["kind"]
    if own:
        from torch2iron_amd import ops
        if kind == "packed":
            return ops.packed_attention(s["q"], s["plan"], s["k_cache"], s["v_cache"], workspace=s["workspace"])
        if kind == "tree":
            return ops.tree_attention(s["q"], s["parents"], s["ctx"], case["hkv"], s["k_cache"], s["v_cache"],
                                      workspace=s["workspace"])
        if kind == "commit":
            path, counts, nxt, context = ops.tree_commit(s["tokens"], s["parents"], s["picks"], s["ctx"], s["k_cache"],
                                                         s["v_cache"])
            return {"path": path, "counts": counts, "next": nxt, "context": context, "k_cache": s["k_cache"],
                    "v_cache": s["v_cache"]}
        lp, entropy, top, ids = ops.token_logprobs(s["logits"], s["tokens"], top_k=case["k"], workspace=s["workspace"])
        return {"logprobs": lp, "entropy": entropy, "top_logprobs": top, "top_ids": ids}
    if kind == "packed":
        return _packed(s)
    if kind == "tree":
        return _tree(s)
    if kind == "commit":
        return _commit(s)
    return _logprobs(s)


# ---- what a pass cannot do without ----

def work(case):
    kind = case["kind"]
    if kind == "packed":
        seqs = _sequences(case)
        rows, slots = sum(a for a, _ in seqs), sum(a + p for a, p in seqs)
        pairs = sum(a * p + a * (a + 1) // 2 for a, p in seqs)
        return {"bytes": 2 * rows * case["hq"] * D * 2 + slots * case["hkv"] * D * 4,
                "flops": 4 * D * case["hq"] * pairs}
    if kind == "tree":
        ctx, n = _contexts(case), case["nodes"]
        # a tree's ancestors depend on the seed: at least the node itself
        pairs = sum(n * (c + 1) for c in ctx)
        return {"bytes": 2 * case["b"] * n * case["hq"] * D * 2 + sum(c + n for c in ctx) * case["hkv"] * D * 4,
                "flops": 4 * D * case["hq"] * pairs}
    if kind == "commit":
        # tokens, parents and picks in, path out; about three rows of a path change their slot
        moved = min(3, case["nodes"] - 1)
        return {"bytes": 16 * case["b"] * case["nodes"] + 2 * moved * case["b"] * case["layers"] * case["hkv"] * D * 4,
                "flops": 0}
    size = TYPES[case["type"]].itemsize
    return {"bytes": case["m"] * (case["v"] * size + 4 + 8 + 8 * case["k"]), "flops": 5 * case["m"] * case["v"]}


# ---- the same in float64, sequence by sequence ----

def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "packed":
        hq, g = case["hq"], case["hq"] // case["hkv"]
        parts, at = [], 0
        for i, (rows, start) in enumerate(zip(s["lens"], s["starts"])):
            out = torch.empty(rows, hq, D, dtype=torch.float64, device=DEV)
            ahead = torch.ones(rows, start + rows, dtype=torch.bool, device=DEV).triu(start + 1)
            for h in range(hq):
                k, v = (s[c][i, h // g, :start + rows].double() for c in ("k_cache", "v_cache"))
                x = (s["q"][at:at + rows, h].double() @ k.T) * D ** -0.5
                x[ahead] = -math.inf
                out[:, h] = torch.softmax(x, -1) @ v
            parts.append(out.view(rows, hq * D))
            at += rows
        return torch.cat(parts)
    if kind == "tree":
        b, n, hq, g = case["b"], case["nodes"], case["hq"], case["hq"] // case["hkv"]
        out = torch.empty(b, n, hq, D, dtype=torch.float64, device=DEV)
        for i, (ctx, parents) in enumerate(zip(s["ctx"].tolist(), s["parents"].tolist())):
            paths = []
            for node in range(n):
                paths.append((paths[parents[node]] if parents[node] >= 0 else []) + [node])
            hidden = torch.ones(n, ctx + n, dtype=torch.bool)
            hidden[:, :ctx] = False
            for node, path in enumerate(paths):
                hidden[node, [ctx + j for j in path]] = False
            hidden = hidden.to(DEV)
            for h in range(hq):
                k, v = (s[c][i, h // g, :ctx + n].double() for c in ("k_cache", "v_cache"))
                x = (s["q"][i, :, h].double() @ k.T) * D ** -0.5
                x[hidden] = -math.inf
                out[i, :, h] = torch.softmax(x, -1) @ v
        return out.view(b * n, hq * D)
    if kind == "commit":
        k, v = s["k_cache"].clone(), s["v_cache"].clone()
        tokens, picks, parents, ctx = (s[c].tolist() for c in ("tokens", "picks", "parents", "ctx"))
        for i in range(case["b"]):
            path = [0]
            while True:
                nxt = [j for j in range(case["nodes"]) if parents[i][j] == path[-1] and tokens[i][j] == picks[i][path[-1]]]
                if not nxt:
                    break
                path.append(nxt[0])
            for to, node in enumerate(path):
                k[:, i, :, ctx[i] + to] = s["k_cache"][:, i, :, ctx[i] + node]
                v[:, i, :, ctx[i] + to] = s["v_cache"][:, i, :, ctx[i] + node]
        return {"path": None, "counts": None, "next": None, "context": None, "k_cache": k.double(), "v_cache": v.double()}
    x = s["logits"].double()
    lp = torch.log_softmax(x, -1)
    best = lp.topk(case["k"], -1).values
    return {"logprobs": lp.gather(1, s["tokens"].long()[:, None])[:, 0], "entropy": -(lp.exp() * lp).sum(-1),
            "top_logprobs": best, "top_ids": None}
