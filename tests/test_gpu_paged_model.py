"""Steps of many requests over a cache in pages, with adapters and drafted tokens, against the CPU oracle.

A greedy token is right when the fp32 oracle, on the same tokens before it, gives it a logit within twice the shift
that bf16 rounding itself causes there of its largest (the oracle's bf16 mode against its fp32 mode); an adapted
request's oracle holds scale B A in its dense weights.  Logits sit no farther from the fp32 oracle's (RMS) than the
bf16-mode oracle's do, within 25 %."""

import pytest
import torch

from oracle import qwen3 as oq
from test_gpu_ragged_model import _check_greedy
from test_gpu_verify import _reference
from torch2iron_amd import model as gm
from torch2iron_amd import ops

pytestmark = pytest.mark.gpu
CAP = 320
BF16 = torch.bfloat16
POOL = 3


@pytest.fixture(scope="module")
def setup(gpu):
    cfg = gm.Qwen3Config(n_layers=2, vocab=2048)
    t = gm.random_qwen3_tensors(cfg, seed=71, weights="centered")
    ocfg = oq.Qwen3Config(**{k: getattr(cfg, k) for k in oq.Qwen3Config.__dataclass_fields__})
    make = lambda: [oq.DenseQwen3(t, ocfg, mode=m, ctx_cap=CAP) for m in ("fp32", "bf16")]  # noqa: E731
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    h, d, inter, rank = cfg.hidden, cfg.head_dim, cfg.intermediate, 12
    q, kv = cfg.n_heads * d, cfg.n_kv_heads * d
    pools, raw = [], []
    for _ in range(cfg.n_layers):
        r = {}
        for name, parts, k, n in (("qkv", 3, h, q + 2 * kv), ("o", 1, q, h), ("gate_up", 2, h, 2 * inter), ("down", 1, inter, h)):
            r[name] = ((rnd(POOL, parts, rank, k) / k ** 0.5).to(BF16), (0.2 * rnd(POOL, n, rank)).to(BF16))
        raw.append(r)
        dev = {n: (a.to(gpu), b.to(gpu)) for n, (a, b) in r.items()}
        pools.append(gm.LayerAdapters(
            qkv=ops.Adapters(*dev["qkv"], scales=torch.tensor([0.5, 1.0, 1.5], device=gpu), widths=[q, kv, kv]),
            o=ops.Adapters(*dev["o"], scales=torch.tensor([0.5, 1.0, 1.5], device=gpu)),
            gate_up=ops.Adapters(*dev["gate_up"], scales=torch.tensor([0.5, 1.0, 1.5], device=gpu), paired=True),
            down=ops.Adapters(*dev["down"], scales=torch.tensor([0.5, 1.0, 1.5], device=gpu))))
    oracles = {-1: make()}
    for i in range(POOL):
        oracles[i] = make()
        for o in oracles[i]:
            for layer, r in zip(o.layers, raw):
                def add(names, key, split):
                    a, b = (x[i].float() for x in r[key])
                    for part, (name, rows) in enumerate(zip(names, split(b))):
                        layer.w[name] = layer.w[name] + 0.5 * (i + 1) * rows @ a[part]
                add(("q_proj", "k_proj", "v_proj"), "qkv", lambda b: b.split((q, kv, kv)))
                add(("o_proj",), "o", lambda b: (b,))
                add(("gate_proj", "up_proj"), "gate_up", lambda b: (b[0::2], b[1::2]))
                add(("down_proj",), "down", lambda b: (b,))
    return cfg, t, oracles, pools


def _model(setup, gpu):
    cfg, t, _, _ = setup
    return gm.Qwen3Model(t, cfg, batch=1, ctx_cap=CAP, device=gpu)


def _i32(gpu, v):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def _serve(gpu, m, cache, prompts, new, draft, chunk, adapters=None, ids=None):
    """Greedy serving of `prompts` in chunks of `chunk` tokens, with `draft(s, emitted)` tokens drafted at each later
    step: the tokens that came out, and the steps it took."""
    n = len(prompts)
    fed, pending, out, steps = [0] * n, [None] * n, [[] for _ in prompts], 0
    while min(map(len, out)) < new:
        rows, drafts, tokens = [], [], []
        for s, p in enumerate(prompts):
            if fed[s] < len(p):
                some = p[fed[s]:fed[s] + chunk].tolist()
                fed[s] += len(some)
                d = 0
            elif len(out[s]) >= new:
                some, d = [], 0
            else:
                drafted = draft(s, len(out[s]))
                some, d = [pending[s]] + drafted, len(drafted)
            rows.append(len(some))
            drafts.append(d)
            tokens += some
            cache.reserve(s, min(len(p) + new + 10, CAP))
        before = cache.lens.tolist()
        batch = gm.PagedBatch(rows, drafts, device=gpu)
        got = m.paged_step(cache, batch, _i32(gpu, tokens), adapters=adapters, adapter_ids=ids)
        counts, nxt, at = got.counts.tolist(), got.next_tokens.tolist(), 0
        for s, (r, d) in enumerate(zip(rows, drafts)):
            if r == 0:
                assert counts[s] == 0 and nxt[s] == -1
            elif fed[s] == len(prompts[s]) or d:
                out[s] += tokens[at + r - d:at + r - d + counts[s]] + [nxt[s]]
                pending[s] = nxt[s]
            at += r
        assert cache.lens.tolist() == [b + r - d + c for b, r, d, c in zip(before, rows, drafts, counts)]
        steps += 1
        assert steps < 80
    return [o[:new] for o in out], steps


@pytest.mark.parametrize("page,chunk", [(16, 1000), (64, 37)], ids=["whole_prompts", "chunks"])
def test_serving_without_adapters(gpu, setup, page, chunk):
    cfg, _, oracles, _ = setup
    m = _model(setup, gpu)
    g = torch.Generator().manual_seed(1)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g) for n in (1, 40, 131, 260)]
    cache = gm.PagedCache(cfg, 4, 60 if page == 16 else 16, CAP // page, gpu, page_slots=page)
    plain, steps = _serve(gpu, m, cache, prompts, 10, lambda s, at: [], chunk)
    for i, p in enumerate(prompts):
        _check_greedy(*oracles[-1], p, plain[i], f"sequence {i}")
    held = cache.free_pages
    for s in range(4):
        cache.release(s)
    assert cache.free_pages == cache.n_pages > held and (cache.table == -1).all()
    # drafted from the plain run, every third token wrong: the same tokens (near-ties aside) in fewer steps
    drafted = lambda s, at: [t if i % 3 else (t + 1) % cfg.vocab for i, t in enumerate(plain[s][at:at + 4], at + 1)]  # noqa: E731
    out, fewer = _serve(gpu, m, cache, prompts, 10, drafted, chunk)
    for i, p in enumerate(prompts):
        _check_greedy(*oracles[-1], p, out[i], f"sequence {i}, drafted")
    assert fewer < steps


@pytest.mark.parametrize("chunk", [1000, 37])
def test_serving_with_adapters(gpu, setup, chunk):
    """Requests of different adapters, and one without, in the same steps; decoding with drafts."""
    cfg, _, oracles, pools = setup
    m = _model(setup, gpu)
    g = torch.Generator().manual_seed(2)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g) for n in (50, 3, 200, 17, 64)]
    ids = [0, 2, -1, 1, 2]
    cache = gm.PagedCache(cfg, 5, 100, CAP // 16, gpu, page_slots=16)
    out, _ = _serve(gpu, m, cache, prompts, 8, lambda s, at: [1, 2] if at % 3 == s % 3 else [], chunk, adapters=pools, ids=_i32(gpu, ids))
    for i, p in enumerate(prompts):
        _check_greedy(*oracles[ids[i]], p, out[i], f"sequence {i}, adapter {ids[i]}")


@pytest.mark.parametrize("lengths", [[30, 9, 20, 1], [150, 200, 90, 120]], ids=["decode_sized", "prompt_gemm"])
def test_logits_with_adapters(gpu, setup, lengths):
    cfg, _, oracles, pools = setup
    m = _model(setup, gpu)
    g = torch.Generator().manual_seed(5)
    prompts = [torch.randint(0, cfg.vocab, (n,), generator=g) for n in lengths]
    ids = [1, -1, 0, 2]
    cache = gm.PagedCache(cfg, 4, 80, CAP // 16, gpu, page_slots=16)
    for s in range(4):
        cache.reserve(s, lengths[s])
    got = m.paged_step(cache, gm.PagedBatch(lengths, device=gpu), torch.cat(prompts).to(torch.int32).to(gpu), adapters=pools,
                       adapter_ids=_i32(gpu, ids))
    logits = got.logits.cpu()
    n_gpu = n_16 = 0.0
    for i, p in enumerate(prompts):
        l32, l16 = (o.prefill(p[None])[0] for o in oracles[ids[i]])
        n_gpu += (logits[i] - l32).pow(2).mean().item()
        n_16 += (l16 - l32).pow(2).mean().item()
    assert n_gpu ** 0.5 <= 1.25 * n_16 ** 0.5, f"logit noise {n_gpu ** 0.5:.4f}, bf16 oracle {n_16 ** 0.5:.4f}"
    # only some projections adapted, and none at all
    some = [gm.LayerAdapters(qkv=a.qkv, down=a.down) for a in pools]
    none = [gm.LayerAdapters() for _ in pools]
    res = []
    for a in (some, none, None):
        for s in range(4):
            cache.release(s)
            cache.reserve(s, lengths[s])
        kw = {} if a is None else dict(adapters=a, adapter_ids=_i32(gpu, ids))
        res.append(m.paged_step(cache, gm.PagedBatch(lengths, device=gpu), torch.cat(prompts).to(torch.int32).to(gpu), **kw).logits)
    assert torch.equal(res[1], res[2]) and not torch.equal(res[0][0], res[2][0])


def test_sampling_follows_the_given_numbers(gpu, setup):
    """Counts and tokens are those of the definition on the step's own logits; what the counts say is in the cache."""
    cfg, _, _, pools = setup
    m = _model(setup, gpu)
    g = torch.Generator().manual_seed(6)
    n, d = 6, 3
    cache = gm.PagedCache(cfg, n, 60, 8, gpu, page_slots=32)
    for s in range(n):
        cache.reserve(s, 200)
    first = gm.PagedBatch([20] * n, device=gpu)
    m.paged_step(cache, first, torch.randint(0, cfg.vocab, (20 * n,), generator=g, dtype=torch.int32).to(gpu))
    batch = gm.PagedBatch([d + 1] * n, [d] * n, device=gpu)
    temps = torch.tensor([0.7, 1.0, 3.0, 0.0, 5.0, 20.0], device=gpu)
    for _ in range(4):
        tokens = torch.randint(0, cfg.vocab, (n * (d + 1),), generator=g, dtype=torch.int32).to(gpu)
        u = torch.rand(n * (d + 1), generator=g).to(gpu)
        q = torch.softmax(torch.randn(n * (d + 1), cfg.vocab, generator=g), -1).to(gpu)
        before = cache.lens.clone()
        got = m.paged_step(cache, batch, tokens, uniforms=u, temperatures=temps, draft_probs=q)
        counts, nxt, lps = _reference(got.logits, batch.head_starts.tolist(), tokens, u, q, temps)
        assert got.counts.tolist() == counts and got.next_tokens.tolist() == nxt
        assert (got.logprobs.cpu().double() - lps).abs().max() < 1e-4
        assert torch.equal(cache.lens, before + 1 + got.counts)


def test_captured_steps(gpu, setup):
    """A decode step with drafts and adapters in one graph, replayed as the caches grow, against eager steps."""
    cfg, _, _, pools = setup
    m = _model(setup, gpu)
    g = torch.Generator().manual_seed(7)
    n = 3
    caches = [gm.PagedCache(cfg, n, 40, CAP // 16, gpu, page_slots=16) for _ in range(2)]
    prompt = torch.randint(0, cfg.vocab, (70,), generator=g, dtype=torch.int32).to(gpu)
    for c in caches:
        for s in range(n):
            c.reserve(s, 200)
        m.paged_step(c, gm.PagedBatch([40, 10, 20], device=gpu), prompt)
    batch = gm.PagedBatch([3, 1, 4], [2, 0, 3], device=gpu)
    tokens, u = torch.zeros(8, dtype=torch.int32, device=gpu), torch.zeros(8, device=gpu)
    temps, ids = torch.tensor([1.0, 0.0, 4.0], device=gpu), _i32(gpu, [0, -1, 2])
    step = lambda c: m.paged_step(c, batch, tokens, uniforms=u, temperatures=temps, adapters=pools, adapter_ids=ids)  # noqa: E731
    state = [x.clone() for x in (caches[0].k, caches[0].v, caches[0].lens)]
    step(caches[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(caches[0])
    for x, y in zip((caches[0].k, caches[0].v, caches[0].lens), state):
        x.copy_(y)
    for i in range(5):
        tokens.copy_(torch.randint(0, cfg.vocab, (8,), generator=g, dtype=torch.int32))
        u.copy_(torch.rand(8, generator=g))
        ids.copy_(torch.randint(-1, POOL, (n,), generator=g, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = step(caches[1])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), f"replay {i}"
        assert torch.equal(caches[0].lens, caches[1].lens) and torch.equal(caches[0].k, caches[1].k)


def test_a_sequence_without_room(gpu, setup):
    """Tokens past the pages that were given out: the sequence ends with -1, the others do not notice."""
    cfg, _, _, _ = setup
    m = _model(setup, gpu)
    g = torch.Generator().manual_seed(8)
    tokens = torch.randint(0, cfg.vocab, (45,), generator=g, dtype=torch.int32).to(gpu)
    res = []
    for slots in (40, 16):
        cache = gm.PagedCache(cfg, 2, 9, 4, gpu, page_slots=16)
        cache.reserve(0, 5)
        cache.reserve(1, slots)
        res.append(m.paged_step(cache, gm.PagedBatch([5, 40], device=gpu), tokens))
    assert res[0].next_tokens[1] >= 0 and res[1].next_tokens[1] == -1
    assert torch.equal(res[0].logits[0], res[1].logits[0]) and torch.isnan(res[1].logits[1]).any()


def test_a_sequence_past_its_part_of_the_table(gpu, setup):
    """Its tokens have no slots at all: NaN logits and the token -1, and the others do not notice."""
    cfg, _, _, _ = setup
    m = _model(setup, gpu)
    g = torch.Generator().manual_seed(9)
    tokens = torch.randint(0, cfg.vocab, (60,), generator=g, dtype=torch.int32).to(gpu)
    res = []
    for first in (3, 59):
        cache = gm.PagedCache(cfg, 2, 8, 4, gpu, page_slots=16)
        for s in range(2):
            cache.reserve(s, 64)
        m.paged_step(cache, gm.PagedBatch([first, 1], device=gpu), tokens[59 - first:])
        k = cache.k.clone()
        u = torch.zeros(6, device=gpu)
        res.append(m.paged_step(cache, gm.PagedBatch([6, 1], [4, 0], device=gpu), tokens[:7], uniforms=u))
    assert (res[0].next_tokens >= 0).all() and torch.isfinite(res[0].logits).all()
    assert res[1].next_tokens[0] == -1 and res[1].counts[0] == 0 and torch.isnan(res[1].logits[:5]).all()
    held = cache.table[0].long()
    assert torch.equal(cache.k[:, held], k[:, held])
    assert res[1].next_tokens[1] == res[0].next_tokens[1] and torch.equal(res[1].logits[5], res[0].logits[5])


def test_refusals(gpu, setup):
    cfg, _, _, pools = setup
    m = _model(setup, gpu)
    cache = gm.PagedCache(cfg, 2, 9, 4, gpu, page_slots=16)
    batch, tokens = gm.PagedBatch([2, 3], [0, 1], device=gpu), _i32(gpu, [1] * 5)
    for s in range(2):
        cache.reserve(s, 10)
    ok = dict(cache=cache, batch=batch, tokens=tokens)
    m.paged_step(**ok)
    u, ids = torch.zeros(3, device=gpu), _i32(gpu, [0, 0])
    before = cache.k.clone(), cache.v.clone(), cache.lens.clone()
    swapped = [gm.LayerAdapters(qkv=a.o) for a in pools]
    for kw in (dict(tokens=tokens[:4]), dict(tokens=tokens.long()), dict(batch=gm.PagedBatch([5], device=gpu)),
               dict(batch=gm.PagedBatch([0, 0], device=gpu), tokens=tokens[:0]), dict(batch=None), dict(cache=None),
               dict(uniforms=u[:2]), dict(temperatures=u[:2]), dict(draft_probs=u), dict(adapters=pools),
               dict(adapters=pools[:1], adapter_ids=ids), dict(adapters=pools, adapter_ids=ids[:1]),
               dict(adapters=swapped, adapter_ids=ids), dict(uniforms=u, temperatures=u), dict(uniforms=u.double()),
               dict(uniforms=u, draft_probs=torch.zeros(3, 64, device=gpu)), dict(uniforms=u.cpu()),
               dict(cache=gm.PagedCache(cfg, 2, 3, CAP // 16 + 1, gpu, page_slots=16)),
               dict(cache=gm.PagedCache(gm.Qwen3Config(n_layers=1, vocab=64), 2, 3, 2, gpu, page_slots=16))):
        with pytest.raises(ValueError):
            m.paged_step(**{**ok, **kw})
    assert all(torch.equal(a, b) for a, b in zip((cache.k, cache.v, cache.lens), before)), "a refused step wrote"


def _used_before(cfg, m, gpu, n_pages):
    """A cache of one sequence whose pages held another request's keys and values before."""
    cache = gm.PagedCache(cfg, 1, n_pages, 6, gpu, page_slots=16)
    g = torch.Generator().manual_seed(40)
    cache.reserve(0, 96)
    m.paged_step(cache, gm.PagedBatch([96], device=gpu), torch.randint(0, cfg.vocab, (96,), generator=g, dtype=torch.int32).to(gpu))
    cache.release(0)
    assert (cache.k[:, :6].float().abs().sum((0, 2, 3, 4)) > 0).all()
    return cache


@pytest.mark.parametrize("start,fed,drafts", [(32, 1, 0), (32, 1, 3), (30, 1, 3), (31, 30, 0)],
                         ids=["token", "drafts", "drafts_over_the_border", "chunk"])
@pytest.mark.parametrize("captured", [False, True], ids=["eager", "captured"])
def test_a_step_without_room_can_be_made_again(gpu, setup, captured, start, fed, drafts):
    """A step that runs past the end of its pages leaves the length as it was; after a reserve the same step, and the one
    after it, have the bits of a run that had room from the start."""
    cfg, _, _, _ = setup
    m = _model(setup, gpu)
    g = torch.Generator().manual_seed(41)
    rnd = lambda n: torch.randint(0, cfg.vocab, (n,), generator=g, dtype=torch.int32).to(gpu)  # noqa: E731
    prompt, tokens, after = rnd(start), rnd(fed + drafts), rnd(1)
    batch, one = gm.PagedBatch([fed + drafts], [drafts], device=gpu), gm.PagedBatch([1], device=gpu)
    u = torch.zeros(drafts + 1, device=gpu)                # every draft of any weight stays
    runs = []
    for slots in (96, 32):
        cache = _used_before(cfg, m, gpu, 6)
        cache.reserve(0, slots)
        assert m.paged_step(cache, gm.PagedBatch([start], device=gpu), prompt).next_tokens[0] >= 0
        step = lambda: m.paged_step(cache, batch, tokens, uniforms=u)  # noqa: E731
        if captured:
            if not runs:
                step()                                     # the workspaces
                cache.lens.fill_(start)
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                got = step()

            def step():
                graph.replay()
                return got

        if slots == 32:
            for _ in range(2):
                got = step()
                assert got.next_tokens.tolist() == [-1] and cache.lens.tolist() == [start]
                torch.cuda.synchronize()
            cache.reserve(0, 96)
        first = [x.clone() for x in step()] + [cache.lens.clone()]
        runs.append(first + list(m.paged_step(cache, one, after)) + [cache.lens.clone()])
    assert runs[0][1].item() >= 0 and runs[0][4].item() == start + fed + runs[0][0].item()
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_a_step_past_the_table_can_be_made_smaller(gpu, setup):
    """Too many tokens for a sequence's part of the table: the length stays, a smaller step fits, and the others go on."""
    cfg, _, _, _ = setup
    m = _model(setup, gpu)
    g = torch.Generator().manual_seed(42)
    tokens = torch.randint(0, cfg.vocab, (64,), generator=g, dtype=torch.int32).to(gpu)
    runs = []
    for too_many in (False, True):
        cache = gm.PagedCache(cfg, 2, 8, 4, gpu, page_slots=16)
        for s in range(2):
            cache.reserve(s, 64)
        m.paged_step(cache, gm.PagedBatch([60, 0], device=gpu), tokens[:60])
        if too_many:
            for n in (5, 70, 5):                           # (70 rows: more than the whole part)
                before = cache.lens.clone()
                many = torch.zeros(n + 1, dtype=torch.int32, device=gpu)
                got = m.paged_step(cache, gm.PagedBatch([n, 1], device=gpu), many)
                assert got.next_tokens[0] == -1 and got.next_tokens[1] >= 0
                assert cache.lens.tolist() == [60, before[1].item() + 1]
        got = m.paged_step(cache, gm.PagedBatch([4, 0], device=gpu), tokens[60:])
        runs.append([got.next_tokens[:1], got.logits, cache.lens[:1]])
        assert cache.lens[0] == 64 and got.next_tokens[0] >= 0
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_tokens_and_adapter_ids_of_another_shape(gpu, setup):
    """As many values in more dimensions are refused, and nothing is written."""
    cfg, _, _, pools = setup
    m = _model(setup, gpu)
    cache = gm.PagedCache(cfg, 2, 9, 4, gpu, page_slots=16)
    batch, tokens, ids = gm.PagedBatch([2, 3], [0, 1], device=gpu), _i32(gpu, [1] * 5), _i32(gpu, [0, 1])
    for s in range(2):
        cache.reserve(s, 10)
    for kw in (dict(tokens=tokens.view(1, 5)), dict(tokens=tokens.view(5, 1)), dict(adapters=pools, adapter_ids=ids.view(1, 2)),
               dict(adapters=pools, adapter_ids=ids.view(2, 1))):
        with pytest.raises(ValueError, match="must be"):
            m.paged_step(cache, batch, **{**dict(tokens=tokens), **kw})
    assert not cache.lens.any() and not cache.k.any() and not cache.v.any()
