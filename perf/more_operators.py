"""What a server of many requests adds to a step, as cases that can be timed and checked.

Three operators of one step that packs prompt chunks, single tokens and drafted tokens of
many requests:

* ``paged_attention``: causal GQA attention of the packed rows over a cache in pages;
* ``verify_drafts``: drafted tokens held to the model's probabilities with given random
  numbers, and the token after them drawn (no drafts: sampling);
* ``adapter_add``: each request's low-rank adapter beside a shared projection.

With ``own`` false ``run`` computes them from elementary torch operations in float32 (the
probabilities, whose running sums have borders finer than that, in float64), rounded once at
the end; with ``own`` true it makes the package's calls.  ``exact`` computes the same from
the definitions in float64, request by request.
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
        # one request's next token: latency
        {"name": "paged_decode_1", "kind": "paged", "hq": 16, "hkv": 8, "page": 16, "n": 0, "lo": 1, "hi": 1,
         "p_lo": 1030, "p_hi": 1030, "singles": 1},
        # the next tokens of a serving batch
        {"name": "paged_decode_32", "kind": "paged", "hq": 16, "hkv": 8, "page": 16, "n": 0, "lo": 1, "hi": 1,
         "p_lo": 409, "p_hi": 4090, "singles": 32},
        # a batch in which every request carries four drafted tokens
        {"name": "paged_drafts_16x5", "kind": "paged", "hq": 32, "hkv": 8, "page": 32, "n": 16, "lo": 5, "hi": 5,
         "p_lo": 901, "p_hi": 4001, "singles": 0},
        # chunks of two long prompts among requests that decode
        {"name": "paged_chunks_24_singles", "kind": "paged", "hq": 32, "hkv": 8, "page": 16, "n": 2, "lo": 509,
         "hi": 701, "p_lo": 2005, "p_hi": 3990, "singles": 24},
        # a late chunk of one long document
        {"name": "paged_1999_after_30001", "kind": "paged", "hq": 32, "hkv": 8, "page": 128, "n": 1, "lo": 1999,
         "hi": 1999, "p_lo": 30001, "p_hi": 30001, "singles": 0},
        # one request with four drafts of a small model: latency
        {"name": "verify_1x4", "kind": "verify", "n": 1, "drafts": 4, "v": VOCAB, "type": "fp32", "probs": True},
        # a batch with drafts looked up in the text (no probabilities), half-precision logits
        {"name": "verify_32x4_bf16", "kind": "verify", "n": 32, "drafts": 4, "v": VOCAB, "type": "bf16",
         "probs": False},
        # a large batch with up to eight drafts of a small model
        {"name": "verify_64x8", "kind": "verify", "n": 64, "drafts": 8, "v": VOCAB, "type": "fp32", "probs": True},
        # decoding: sixteen requests, each with an adapter of its own, beside the fused q|k|v projection
        {"name": "adapters_16_qkv", "kind": "adapters", "k": 1024, "widths": "2048,1024,1024", "paired": False,
         "rank": 16, "pool": 32, "requests": 16, "lo": 1, "hi": 1},
        # short prompts beside the paired gate and up projection, SwiGLU behind it
        {"name": "adapters_331_gate_up", "kind": "adapters", "k": 2048, "widths": "12288", "paired": True,
         "rank": 64, "pool": 8, "requests": 7, "lo": 5, "hi": 150},
        # long prompts beside the down projection
        {"name": "adapters_4001_down", "kind": "adapters", "k": 6144, "widths": "2048", "paired": False,
         "rank": 32, "pool": 8, "requests": 3, "lo": 700, "hi": 2100},
        # a full prompt batch beside the fused q|k|v projection
        {"name": "adapters_8192_qkv", "kind": "adapters", "k": 2048, "widths": "4096,1024,1024", "paired": False,
         "rank": 16, "pool": 16, "requests": 16, "lo": 512, "hi": 512},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case of the listed ranges."""
    kind = rng.choice(["paged", "paged", "paged", "verify", "verify", "adapters", "adapters"])
    if kind == "paged":
        hkv, g = rng.choice([(8, 2), (8, 4), (8, 1), (4, 8), (2, 7), (8, 3)])
        page = rng.choice([16, 16, 32, 64, 128, 256])
        form = rng.choice(["decode", "drafts", "chunks", "one"])
        c = {"kind": kind, "hq": hkv * g, "hkv": hkv, "page": page, "n": 0, "lo": 1, "hi": 1, "singles": 0}
        if form == "decode":
            c["singles"] = _log(rng, 1, 64)
            p_hi = _log(rng, 1, min(32000, 130000 // c["singles"]))
        elif form == "drafts":
            c["n"] = _log(rng, 1, 32)
            c["hi"] = rng.randrange(2, 10)
            c["lo"] = rng.randrange(1, c["hi"] + 1)
            p_hi = _log(rng, 1, min(32000, 90000 // c["n"]))
        elif form == "chunks":
            c["n"] = rng.choice([2, 3, 7, 16])
            c["singles"] = rng.choice([0, rng.randrange(1, 25)])
            c["hi"] = _log(rng, 10, 900 if c["n"] < 4 else 300)
            c["lo"] = rng.randrange(1, c["hi"] + 1)
            p_hi = rng.choice([0, _log(rng, 1, 4000)])
        else:
            c["n"] = 1
            c["lo"] = c["hi"] = _log(rng, 10, 1900)
            p_hi = rng.choice([0, _log(rng, 1, 28000)])
        return {**c, "p_lo": rng.randrange(0, p_hi + 1), "p_hi": p_hi}
    if kind == "verify":
        drafts = rng.choice([0, 1, 2, 4, 5, 8])
        return {"kind": kind, "n": _log(rng, 1, 570 // (drafts + 1)), "drafts": drafts,
                "v": rng.choice([VOCAB, VOCAB, 4096, _log(rng, 1000, 150000)]),
                "type": rng.choice(["fp32", "fp32", "bf16", "fp16"]), "probs": rng.random() < 0.5}
    form = rng.choice(["qkv", "one", "paired"])
    k = rng.choice([1024, 2048, 4096, 6144])
    widths = {"qkv": rng.choice(["2048,1024,1024", "4096,1024,1024"]), "one": rng.choice(["1024", "2048", "4096"]),
              "paired": rng.choice(["6144", "12288"])}[form]
    requests = _log(rng, 1, 64)
    hi = rng.choice([1, _log(rng, 1, max(1, (3000 if form == "paired" else 8000) // requests))])
    return {"kind": kind, "k": k, "widths": widths, "paired": form == "paired", "rank": rng.choice([8, 16, 32, 64, 128, 20]),
            "pool": rng.choice([1, 4, 16, 64]), "requests": requests, "lo": rng.randrange(1, hi + 1), "hi": hi}


# ---- inputs, from the seed alone ----

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, device=DEV, generator=g).to(BF16)


def _spread(n, lo, hi):
    """n whole numbers from lo to hi, spread over their logarithm."""
    return [round(lo * (hi / lo) ** (i / (n - 1))) if n > 1 else hi for i in range(n)]


def _sequences(case):
    """(rows, slots before them) of each request: rows spread over their logarithm, earlier
    slots evenly; then the requests of one row."""
    n, p_lo, p_hi, s = case["n"], case["p_lo"], case["p_hi"], case["singles"]
    some = [(rows, p_hi - (p_hi - p_lo) * i // max(n - 1, 1)) for i, rows in enumerate(_spread(n, case["lo"], case["hi"]))]
    return some + [(1, p_hi - (p_hi - p_lo) * i // max(s - 1, 1)) for i in range(s)]


def _drafted(case):
    """Drafted tokens of each request: half of them as many as there may be, the others fewer."""
    d = case["drafts"]
    return [d if i % 2 == 0 else max(0, d - 1 - i // 2 % max(d, 1)) for i in range(case["n"])]


def _requests(case):
    """(rows, whether it has an adapter) of each request; of five one has none."""
    return [(rows, i % 5 != 4) for i, rows in enumerate(_spread(case["requests"], case["lo"], case["hi"]))]


def _place(s, lens):
    """Where each packed row stands in the padded batch, for the plain forms."""
    seq = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens))
    first = torch.tensor([0] + lens).cumsum(0)[:-1]
    s["row_seq"], s["row_t"], s["longest"] = seq.to(DEV), (torch.arange(len(seq)) - first[seq]).to(DEV), max(lens)


def _prepare_paged(case, seed, g, s):
    seqs = _sequences(case)
    random.Random(seed).shuffle(seqs)
    page = case["page"]
    lens, starts = [a for a, _ in seqs], [b for _, b in seqs]
    need = [-(-(a + b) // page) for a, b in seqs]
    # pages as a server has given them out: in no order, a few of them free
    order = torch.randperm(sum(need) + 5, device=DEV, generator=g).to(torch.int32)
    table = torch.full((len(seqs), max(need) + 2), -1, dtype=torch.int32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    s["table"] = table
    s["row_starts"] = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    s["ctx"] = torch.tensor(starts, dtype=torch.int32).to(DEV)
    s["lens"], s["starts"] = lens, starts
    s["q"] = _normal(g, sum(lens), case["hq"], D)
    s["k_pages"], s["v_pages"] = (_normal(g, order.numel(), case["hkv"], page, D) for _ in range(2))
    if own:
        from torch2iron_amd import ops
        s["plan"] = ops.PagedPlan(sum(lens), s["row_starts"], s["ctx"], s["table"], case["hq"], case["hkv"], page)
        s["workspace"] = ops.Workspace()
    else:
        _place(s, lens)
        s["pages"] = max(need)


def _prepare_verify(case, seed, g, s):
    n, v = case["n"], case["v"]
    drafted = _drafted(case)
    random.Random(seed).shuffle(drafted)
    lens = [d + 1 for d in drafted]
    m = sum(lens)

    def noise():
        return torch.randn(m, v, device=DEV, generator=g)

    # logits as models give them: a few likely tokens a row over a long tail
    x = noise() * 2
    hot = (torch.randint(0, v, (m, 1), device=DEV, generator=g) + torch.arange(6, device=DEV) * (v // 6)) % v
    x.scatter_(1, hot, 10 + 3 * torch.randn(m, 6, device=DEV, generator=g))
    draft = x + 0.7 * noise()
    s["logits"] = x.to(TYPES[case["type"]])
    # the token after a row: drawn from the draft's distribution (the largest of its logits and Gumbel noise)
    u = torch.rand(m, v, device=DEV, generator=g).clamp_(1e-10, 1 - 1e-7)
    after = (draft - torch.log(-torch.log(u))).argmax(-1).to(torch.int32)
    s["tokens"] = torch.roll(after, 1)
    s["probs"] = torch.softmax(draft, -1) if case["probs"] else None
    s["uniforms"] = torch.rand(m, device=DEV, generator=g)
    t = 0.6 + 0.6 * torch.rand(n, device=DEV, generator=g)
    s["temperatures"] = torch.where(torch.arange(n, device=DEV) % 8 == 7, 0.0, t)       # of eight one is greedy
    s["row_starts"] = torch.tensor([0] + lens).cumsum(0).to(torch.int32).to(DEV)
    s["lens"] = lens
    if own:
        from torch2iron_amd import ops
        s["workspace"] = ops.Workspace()
    else:
        _place(s, lens)


def _prepare_adapters(case, seed, g, s):
    widths = [int(w) for w in case["widths"].split(",")]
    parts, n, k, r = 2 if case["paired"] else len(widths), sum(widths), case["k"], case["rank"]
    reqs = _requests(case)
    rng = random.Random(seed)
    rng.shuffle(reqs)
    lens, m = [a for a, _ in reqs], sum(a for a, _ in reqs)
    which = [rng.randrange(case["pool"]) if has else -1 for _, has in reqs]
    s["which"], s["lens"], s["widths"] = which, lens, widths
    s["ids"] = torch.repeat_interleave(torch.tensor(which, dtype=torch.int32), torch.tensor(lens)).to(DEV)
    s["x"], s["y"] = _normal(g, m, k), _normal(g, m, n)
    s["a"] = (torch.randn(case["pool"], parts, r, k, device=DEV, generator=g) / math.sqrt(k)).to(BF16)
    s["b"] = (torch.randn(case["pool"], n, r, device=DEV, generator=g) / math.sqrt(r)).to(BF16)
    s["scales"] = 0.25 + torch.rand(case["pool"], device=DEV, generator=g)
    if own:
        from torch2iron_amd import ops
        s["adapters"] = ops.Adapters(s["a"], s["b"], s["scales"], widths=None if case["paired"] else widths,
                                     paired=case["paired"])
        s["plan"] = ops.AdapterPlan(s["ids"], case["pool"])
        s["workspace"] = ops.Workspace()
    else:
        _place(s, lens)
        s["of"] = torch.tensor(which).to(DEV)


def prepare(case, seed):
    s = {"case": case}
    {"paged": _prepare_paged, "verify": _prepare_verify, "adapters": _prepare_adapters}[case["kind"]](case, seed, _gen(seed), s)
    return s


# ---- the operators ----

def _paged(s):
    case = s["case"]
    hq, hkv, b, t = case["hq"], case["hkv"], len(s["lens"]), s["longest"]
    pages = s["table"][:, :s["pages"]].clamp(min=0).long()
    keys = s["pages"] * case["page"]
    k, v = (s[c][pages].transpose(1, 2).reshape(b, hkv, keys, D).float() for c in ("k_pages", "v_pages"))
    q = torch.zeros(b, t, hq, D, dtype=torch.float32, device=DEV)
    q[s["row_seq"], s["row_t"]] = s["q"].float()
    q = q.view(b, t, hkv, hq // hkv, D).permute(0, 2, 3, 1, 4).reshape(b, hkv, -1, D)      # rows (head, t)
    pos = s["ctx"].long()[:, None] + torch.arange(t, device=DEV)
    seen = torch.arange(keys, device=DEV) <= pos[:, :, None]                               # [B, T, K]
    seen = seen[:, None].expand(b, hq // hkv, t, keys).reshape(b, 1, -1, keys)
    x = torch.matmul(q, k.transpose(-1, -2).contiguous()) / math.sqrt(D)
    x = x.masked_fill(~seen, -math.inf)
    w = torch.exp(x - x.amax(-1, keepdim=True))
    # what a page holds behind the last slot has no weight, whatever it is
    o = torch.matmul(w, v) / w.sum(-1, keepdim=True)
    o = o.view(b, hq, t, D).transpose(1, 2)[s["row_seq"], s["row_t"]]
    return o.reshape(-1, hq * D).to(BF16)


def _first(hit):
    """The first true place of each row."""
    at = torch.arange(hit.shape[-1], device=DEV)
    return torch.where(hit, at, hit.shape[-1]).amin(-1)


def _verify(s):
    starts = s["row_starts"].long()
    first, last = starts[:-1], starts[1:] - 1
    m, v = s["logits"].shape
    temp = s["temperatures"].double()
    greedy = (temp <= 0)[s["row_seq"]]
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    y = (x - top) / torch.where(temp > 0, temp, 1.0)[s["row_seq"]][:, None]
    e = torch.exp(y)
    z = e.sum(-1, keepdim=True)
    best = _first(x == top)                                        # the lowest of equal maxima
    # each row's draft, and whether it is taken
    rows = torch.arange(m, device=DEV)
    has = rows < last[s["row_seq"]]
    draft = s["tokens"].long().roll(-1)
    p = e.gather(1, draft[:, None])[:, 0] / z[:, 0]
    q = 1.0 if s["probs"] is None else s["probs"].gather(1, draft[:, None])[:, 0].double()
    taken = torch.where(greedy, draft == best, s["uniforms"].double() * q < p) & has
    # drafts taken before the first that is not
    pad = torch.zeros(len(s["lens"]), s["longest"], dtype=torch.bool, device=DEV)
    pad[s["row_seq"], s["row_t"]] = taken
    counts = pad.long().cumprod(-1).sum(-1)
    # the row after which the next token comes, and the weights that it is drawn by
    row = first + counts
    w = e[row] / z[row]
    if s["probs"] is None:
        less = torch.zeros_like(w).scatter_(1, draft[row][:, None], 1.0)
    else:
        less = s["probs"][row].double()
    rest = torch.where(has[row][:, None], (w - less).clamp(min=0), w)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
    c = rest.cumsum(-1)
    drawn = _first(c > s["uniforms"].double()[last][:, None] * c[:, -1:])
    nxt = torch.where(greedy[row], best[row], drawn)
    # the log probability of what came out after each row
    out = torch.where(rows == row[s["row_seq"]], nxt[s["row_seq"]], draft)
    lp = y.gather(1, out[:, None])[:, 0] - torch.log(z[:, 0])
    lp = torch.where(rows <= row[s["row_seq"]], lp, 0.0)
    return {"counts": counts.to(torch.int32), "next": nxt.to(torch.int32), "logprobs": lp.float()}


def _adapters(s):
    case, b, t = s["case"], len(s["lens"]), s["longest"]
    some = (s["of"] >= 0)[:, None, None]
    of = s["of"].clamp(min=0)
    x = torch.zeros(b, t, case["k"], dtype=torch.float32, device=DEV)
    x[s["row_seq"], s["row_t"]] = s["x"].float()
    parts = s["a"].shape[1]
    a = s["a"][of].float()
    h = [torch.matmul(x, a[:, i].transpose(1, 2).contiguous()) for i in range(parts)]
    bt = s["b"][of].float().transpose(1, 2)
    cols = [bt[:, :, i::2] for i in range(2)] if case["paired"] else bt.split(s["widths"], 2)
    scale = s["scales"][of][:, None, None]
    add = [torch.where(some, torch.matmul(u, c.contiguous()) * scale, 0.0)[s["row_seq"], s["row_t"]] for u, c in zip(h, cols)]
    y = s["y"].float()
    if case["paired"]:
        gate, up = y[:, 0::2] + add[0], y[:, 1::2] + add[1]
        return (gate / (1 + torch.exp(-gate)) * up).to(BF16)
    return (y + torch.cat(add, 1)).to(BF16)


def run(s):
    kind = s["case"]["kind"]
    if own:
        from torch2iron_amd import ops
        if kind == "paged":
            return ops.paged_attention(s["q"], s["plan"], s["k_pages"], s["v_pages"], workspace=s["workspace"])
        if kind == "verify":
            counts, nxt, lp = ops.verify_drafts(s["logits"], s["row_starts"], s["tokens"], s["uniforms"],
                                                draft_probs=s["probs"], temperatures=s["temperatures"],
                                                workspace=s["workspace"])
            return {"counts": counts, "next": nxt, "logprobs": lp}
        out = torch.empty(s["y"].shape[0], s["y"].shape[1] // (2 if s["case"]["paired"] else 1), dtype=BF16, device=DEV)
        return ops.adapter_add(s["y"], s["x"], s["adapters"], s["plan"], out=out, swiglu=s["case"]["paired"],
                               workspace=s["workspace"])
    return {"paged": _paged, "verify": _verify, "adapters": _adapters}[kind](s)


# ---- what a pass cannot do without ----

def work(case):
    kind = case["kind"]
    if kind == "paged":
        seqs = _sequences(case)
        rows, slots = sum(a for a, _ in seqs), sum(a + p for a, p in seqs)
        pairs = sum(a * p + a * (a + 1) // 2 for a, p in seqs)
        return {"bytes": 2 * rows * case["hq"] * D * 2 + slots * case["hkv"] * D * 4,
                "flops": 4 * D * case["hq"] * pairs}
    if kind == "verify":
        m, size = case["n"] + sum(_drafted(case)), TYPES[case["type"]].itemsize
        # every row's logits; the draft's probabilities where one was refused (about half of the requests that have any)
        refused = sum(d > 0 for d in _drafted(case)) // 2 if case["probs"] else 0
        return {"bytes": m * (case["v"] * size + 12) + refused * case["v"] * 4 + case["n"] * 16, "flops": 4 * m * case["v"]}
    widths = [int(w) for w in case["widths"].split(",")]
    parts, n, k, r = 2 if case["paired"] else len(widths), sum(widths), case["k"], case["rank"]
    reqs = _requests(case)
    m, rows = sum(a for a, _ in reqs), sum(a for a, has in reqs if has)
    adapters = min(case["pool"], sum(has for _, has in reqs))
    out = n // 2 if case["paired"] else n
    return {"bytes": 2 * (rows * k + m * (n + out) + adapters * r * (parts * k + n)) + 4 * m,
            "flops": 2 * rows * r * (parts * k + n)}


# ---- the same in float64, request by request ----

def _exact_paged(case, s):
    hq, g, page = case["hq"], case["hq"] // case["hkv"], case["page"]
    parts, at = [], 0
    for i, (rows, start) in enumerate(zip(s["lens"], s["starts"])):
        slots = torch.arange(start + rows, device=DEV)
        where, inside = s["table"][i].long()[slots // page], slots % page
        out = torch.empty(rows, hq, D, dtype=torch.float64, device=DEV)
        ahead = torch.ones(rows, start + rows, dtype=torch.bool, device=DEV).triu(start + 1)
        for h in range(hq):
            k, v = (s[c][where, h // g, inside].double() for c in ("k_pages", "v_pages"))
            x = (s["q"][at:at + rows, h].double() @ k.T) * D ** -0.5
            x[ahead] = -math.inf
            out[:, h] = torch.softmax(x, -1) @ v
        parts.append(out.view(rows, hq * D))
        at += rows
    return torch.cat(parts)


def _exact_verify(case, s):
    logprobs, at = torch.zeros(sum(s["lens"]), dtype=torch.float64, device=DEV), 0
    tokens, uniforms, temps = s["tokens"].tolist(), s["uniforms"].double().tolist(), s["temperatures"].double().tolist()
    for n, temp in zip(s["lens"], temps):
        for row in range(at, at + n):
            x = s["logits"][row].double()
            lp = torch.log_softmax(x / temp if temp > 0 else x, -1)
            best = int((x == x.max()).nonzero()[0])
            if row + 1 < at + n:
                y = tokens[row + 1]
                q = 1.0 if s["probs"] is None else float(s["probs"][row, y].double())
                ok = y == best if temp <= 0 else uniforms[row] * q < float(lp[y].exp())
                if ok:
                    logprobs[row] = lp[y]
                    continue
                w = lp.exp()
                if s["probs"] is None:
                    w[y] = 0
                else:
                    w = (w - s["probs"][row].double()).clamp(min=0)
                w = w if float(w.sum()) > 0 else lp.exp()
            else:
                w = lp.exp()
            c = w.cumsum(0)
            drawn = best if temp <= 0 else int((c > uniforms[at + n - 1] * c[-1]).nonzero()[0])
            logprobs[row] = lp[drawn]
            break
        at += n
    return {"counts": None, "next": None, "logprobs": logprobs}


def _exact_adapters(case, s):
    parts, at = [], 0
    for which, rows in zip(s["which"], s["lens"]):
        y = s["y"][at:at + rows].double()
        if which >= 0:
            x, scale = s["x"][at:at + rows].double(), float(s["scales"][which].double())
            a, b = s["a"][which].double(), s["b"][which].double()
            if case["paired"]:
                for i in range(2):
                    y[:, i::2] += scale * (x @ a[i].T) @ b[i::2].T
            else:
                col = 0
                for i, w in enumerate(s["widths"]):
                    y[:, col:col + w] += scale * (x @ a[i].T) @ b[col:col + w].T
                    col += w
        parts.append(torch.nn.functional.silu(y[:, 0::2]) * y[:, 1::2] if case["paired"] else y)
        at += rows
    return torch.cat(parts)


def exact(case, seed):
    s = prepare(case, seed)
    return {"paged": _exact_paged, "verify": _exact_verify, "adapters": _exact_adapters}[case["kind"]](case, s)
