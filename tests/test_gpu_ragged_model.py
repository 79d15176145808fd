"""Prompts of different lengths, scoring and drafted trees through the model, against the CPU oracle.

A token that the model picks is right when the fp32 oracle, on the same tokens before it, gives it a
logit within twice the shift that bf16 rounding itself causes there of its largest (the oracle's bf16
mode against its fp32 mode): a near-tie.  Log probabilities and entropies sit no farther from the fp32
oracle's (RMS) than the bf16-mode oracle's do, within 25 %, as the model's logits elsewhere."""

import pytest
import torch

from oracle import qwen3 as oq
from torch2iron_amd import model as gm
from torch2iron_amd import ops

pytestmark = pytest.mark.gpu
CAP = 320


@pytest.fixture(scope="module")
def setup(gpu):
    cfg = gm.Qwen3Config(n_layers=2, vocab=2048)
    t = gm.random_qwen3_tensors(cfg, seed=61, weights="centered")
    ocfg = oq.Qwen3Config(**{k: getattr(cfg, k) for k in oq.Qwen3Config.__dataclass_fields__})
    o32, o16 = (oq.DenseQwen3(t, ocfg, mode=m, ctx_cap=CAP) for m in ("fp32", "bf16"))
    return cfg, t, o32, o16


def _prompts(cfg, lengths, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, cfg.vocab, (n,), generator=g) for n in lengths]


def _check_greedy(o32, o16, prompt, tokens, what):
    """Every token of ``tokens`` follows its history as greedy decode would, near-ties aside."""
    forced = torch.as_tensor(tokens)[None]
    l32 = o32.forced_logits(prompt[None], forced[:, :-1])[0]
    l16 = o16.forced_logits(prompt[None], forced[:, :-1])[0]
    for s, tok in enumerate(tokens):
        noise = (l16[s] - l32[s]).abs().max().item()
        gap = (l32[s].max() - l32[s, tok]).item()
        assert gap <= 2.0 * noise, f"{what}, step {s}: {gap:.3f} below the best, bf16 noise {noise:.3f}"


@pytest.mark.parametrize("lengths", [[1, 37, 64, 9], [5], [300, 17, 1, 260, 131]], ids=["short", "one", "prompt_gemm"])
def test_generate_from_prompts_of_different_lengths(gpu, setup, lengths):
    cfg, t, o32, o16 = setup
    m = gm.Qwen3Model(t, cfg, batch=len(lengths), ctx_cap=CAP, device=gpu)
    prompts = _prompts(cfg, lengths, 1)
    got = m.generate(prompts, 12)
    again = m.generate([p.tolist() for p in prompts], 12, use_graph=False)
    assert torch.equal(got, again), "graph replay differs from eager launches"
    assert m.positions.tolist() == [n + 11 for n in lengths]
    logits = m.prefill_packed(prompts, want_logits=True).cpu()
    n_gpu = n_16 = 0.0
    for i, p in enumerate(prompts):
        _check_greedy(o32, o16, p, got[i].tolist(), f"prompt of {len(p)}")
        l32, l16 = o32.prefill(p[None])[0], o16.prefill(p[None])[0]
        n_gpu += (logits[i] - l32).pow(2).mean().item()
        n_16 += (l16 - l32).pow(2).mean().item()
    assert n_gpu ** 0.5 <= 1.25 * n_16 ** 0.5, f"logit noise {n_gpu ** 0.5:.4f}, bf16 oracle {n_16 ** 0.5:.4f}"


def test_equal_lengths_fill_the_cache_as_the_batch_pass(gpu, setup):
    """Layer 0's K and V are the same bits; the first tokens those of the batch pass (near-ties aside)."""
    cfg, t, o32, o16 = setup
    prompts = _prompts(cfg, [200, 200, 200], 2)
    a, b = (gm.Qwen3Model(t, cfg, batch=3, ctx_cap=CAP, device=gpu) for _ in range(2))
    a.prefill(torch.stack(prompts).to(gpu))
    b.prefill_packed(prompts)
    assert torch.equal(a.k_cache[0, :, :, :200], b.k_cache[0, :, :, :200])
    assert torch.equal(a.v_cache[0, :, :, :200], b.v_cache[0, :, :, :200])
    for i, p in enumerate(prompts):
        _check_greedy(o32, o16, p, [int(b.tokens[i])], f"sequence {i}")


def test_score(gpu, setup):
    cfg, t, o32, o16 = setup
    lengths = [1, 70, 2, 251]
    m = gm.Qwen3Model(t, cfg, batch=4, ctx_cap=CAP, device=gpu)
    prompts = _prompts(cfg, lengths, 3)
    sq = {"lp": [0.0, 0.0], "entropy": [0.0, 0.0]}
    for p, s in zip(prompts, m.score(prompts, top_k=6)):
        n = len(p)
        assert s.logprobs.shape == (n - 1,) and s.entropy.shape == (n,) and s.top_ids.shape == (n, 6)
        l32, l16 = (torch.log_softmax(o.forced_logits(p[None, :1], p[None, 1:])[0].double(), -1) for o in (o32, o16))
        ent = [-(x.exp() * x).sum(-1) for x in (l32, l16)]
        at = [x[:-1].gather(1, p[1:, None])[:, 0] for x in (l32, l16)]
        for key, got, ref in (("lp", s.logprobs, at), ("entropy", s.entropy, ent)):
            sq[key][0] += (got.cpu().double() - ref[0]).pow(2).sum().item()
            sq[key][1] += (ref[1] - ref[0]).pow(2).sum().item()
        top, ids = s.top_logprobs.cpu(), s.top_ids.cpu().long()
        assert (top[:, :-1] >= top[:, 1:]).all()
        noise = (l16 - l32).abs().amax(-1, keepdim=True)
        assert ((top - l32.gather(1, ids)).abs() <= 2 * noise).all()
        assert ((l32.amax(-1) - l32.gather(1, ids[:, :1])[:, 0]) <= 2 * noise[:, 0]).all()
    for key, (gpu_sq, ref_sq) in sq.items():
        assert gpu_sq ** 0.5 <= 1.25 * ref_sq ** 0.5, f"{key}: {gpu_sq ** 0.5:.4f} against {ref_sq ** 0.5:.4f}"


def _tree(true, emitted, vocab, g):
    """A drafted tree of 11 nodes that holds up to four of the tokens to come on a winding path among
    decoys: nodes 2, 5, 6, 10 under 0, 2, 5, 6."""
    tokens = torch.randint(0, vocab, (11,), generator=g)
    parents = torch.tensor([-1, 0, 0, 1, 2, 2, 5, 5, 3, 6, 6], dtype=torch.int32)
    for at, node in enumerate((2, 5, 6, 10)):
        if emitted + at < len(true):
            tokens[node] = true[emitted + at]
    return tokens.to(torch.int32), parents


def test_verified_trees_decode_as_greedy(gpu, setup):
    """Decoding by drafted trees: tokens, positions and the cache are those of greedy decode; plain decode
    goes on from them; a sequence without nodes waits; one without room stays."""
    cfg, t, o32, o16 = setup
    lengths, new = [1, 40, 131], 20
    m = gm.Qwen3Model(t, cfg, batch=3, ctx_cap=CAP, device=gpu)
    prompts = _prompts(cfg, lengths, 4)
    true = m.generate(prompts, new + 8).tolist()
    m.history = None
    m.prefill_packed(prompts)
    out = [[int(x)] for x in m.tokens.tolist()]
    g = torch.Generator().manual_seed(5)
    steps = accepted = 0
    while min(map(len, out)) < new:
        trees = [_tree(true[i], len(out[i]), cfg.vocab, g) for i in range(3)]
        counts = torch.tensor([11, 11 if steps != 1 else 0, 7], dtype=torch.int32)
        before = m.positions.tolist()
        got, n = m.verify_tree(torch.stack([a for a, _ in trees]).to(gpu), torch.stack([b for _, b in trees]).to(gpu),
                               node_counts=counts.to(gpu))
        got, n = got.tolist(), n.tolist()
        for i in range(3):
            assert (n[i] == 0) == (int(counts[i]) == 0)
            assert got[i][n[i]:] == [-1] * (11 - n[i]) and min(got[i][:n[i]], default=0) >= 0
            out[i] += got[i][:n[i]]
        assert m.positions.tolist() == [b + k for b, k in zip(before, n)]
        assert m.tokens.tolist() == [o[-1] for o in out]
        accepted += sum(k - 1 for k in n if k)
        steps += 1
        assert steps < 60
    assert accepted >= 3 * new // 3, f"{accepted} drafted tokens accepted in {steps} steps"
    for _ in range(4):                     # plain decode steps on the same state
        m.forward_step()
        ops.greedy_advance(m.keys, m.tokens, m.positions, None, m.step)
        for o, x in zip(out, m.tokens.tolist()):
            o.append(x)
    for i, p in enumerate(prompts):
        _check_greedy(o32, o16, p, out[i], f"sequence {i}")
    # no room for the nodes: nothing moves
    m.positions[1] = CAP - 3
    state = m.positions.clone(), m.tokens.clone(), m.k_cache[:, 1].clone()
    tok, par = _tree(true[1], 0, cfg.vocab, g)
    _, n = m.verify_tree(tok.repeat(3, 1).to(gpu), par.repeat(3, 1).to(gpu))
    assert n.tolist()[1] == 0 and m.positions[1] == state[0][1] and m.tokens[1] == state[1][1]
    assert torch.equal(m.k_cache[:, 1], state[2])
    with pytest.raises(ValueError):
        m.verify_tree(tok.repeat(2, 1).to(gpu), par.repeat(3, 1).to(gpu))
    with pytest.raises(ValueError):
        m.verify_tree(tok.repeat(3, 1).to(gpu).long(), par.repeat(3, 1).to(gpu))


def test_verify_tree_replayed_from_a_graph(gpu, setup):
    cfg, t, _, _ = setup
    a, b = (gm.Qwen3Model(t, cfg, batch=3, ctx_cap=CAP, device=gpu) for _ in range(2))
    prompts = _prompts(cfg, [33, 2, 70], 6)
    g = torch.Generator().manual_seed(7)
    tok = torch.zeros(3, 11, dtype=torch.int32, device=gpu)
    par = _tree([], 0, cfg.vocab, g)[1].repeat(3, 1).to(gpu)
    for m in (a, b):
        m.prefill_packed(prompts)
    state = [x.clone() for x in (a.tokens, a.positions, a.k_cache, a.v_cache)]
    a.verify_tree(tok, par)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = a.verify_tree(tok, par)
    for x, y in zip((a.tokens, a.positions, a.k_cache, a.v_cache), state):
        x.copy_(y)
    for _ in range(4):
        tok.copy_(torch.randint(0, cfg.vocab, (3, 11), generator=g, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = b.verify_tree(tok, par)
        assert torch.equal(res[0], want[0]) and torch.equal(res[1], want[1])
        assert torch.equal(a.positions, b.positions) and torch.equal(a.k_cache, b.k_cache)


def test_prompt_refusals(gpu, setup):
    cfg, t, _, _ = setup
    m = gm.Qwen3Model(t, cfg, batch=2, ctx_cap=16, device=gpu)
    ok = torch.zeros(3, dtype=torch.int64)
    for bad in ([ok], [ok, ok[:0]], [ok, torch.zeros(17, dtype=torch.int64)], [ok, ok - 1], [ok, ok + cfg.vocab],
                [ok, ok[None]]):
        with pytest.raises(ValueError):
            m.prefill_packed(bad)
        with pytest.raises(ValueError):
            m.score(bad)
    with pytest.raises(ValueError):
        m.generate([ok, ok[:1]], 4, prompt_mode="decode")
    with pytest.raises(ValueError):
        m.generate([ok, torch.zeros(14, dtype=torch.int64)], 4)
