"""The batch operators together, as a server uses them: a ragged prompt step, then decode steps of the
whole batch, through a small W4A16 model's layers; every sequence against the one-sequence runner."""
import math

import pytest
import torch
import torch.nn.functional as F

from nanoserve_amd.qwen import Qwen2Runner, Qwen2Shape
from oracle import decode_ref

pytestmark = pytest.mark.gpu


def _batch_forward(r, x, pools, pages, lens, q_start, shared, work):
    """Logits of every token row of a batch: the layers of Qwen2Runner.forward with the paged operators
    in place of one sequence's."""
    s, k, pending = r.shape, r.k, None
    for li, L in enumerate(r.layers):
        h = k.rmsnorm(x, pending, L["ln_in"], s.eps)
        kp, vp = pools[0][li], pools[1][li]
        q = k.paged_append(k.w4_linear(h, *L["wqkv"]), L["bqkv"], r.inv_freq, pages, lens, kp, vp, s.heads,
                           q_start=q_start)
        a = k.paged_attention(q, kp, vp, pages, lens, s.heads, q_start=q_start, shared=shared, work=work)
        h = k.rmsnorm(x, k.w4_linear(a, *L["wo"]), L["ln_post"], s.eps)
        pending = k.w4_linear(k.w4_linear_swiglu(h, *L["wgu"]), *L["wd"])
    return F.linear(k.rmsnorm(x, pending, r.final_norm, s.eps), r.lm_head)


@pytest.mark.parametrize("prefix", [0, 40])
def test_batch_matches_single_sequences(kernels, prefix):
    shape = Qwen2Shape(layers=2, hidden=512, heads=4, kv_heads=2, intermediate=1024, vocab=2000)
    r = Qwen2Runner.random(shape, seed=3, kernels=kernels)
    g = torch.Generator().manual_seed(prefix)
    common = torch.randint(0, shape.vocab, (prefix,), generator=g)
    prompts = [torch.cat([common, torch.randint(0, shape.vocab, (n,), generator=g)]).cuda() for n in (5, 33, 1, 90)]
    B, steps, page = len(prompts), 6, 16
    width = (max(map(len, prompts)) + steps) // page + 1
    pools = torch.zeros(2, shape.layers, B * width, shape.kv_heads, page, shape.head_dim, dtype=torch.bfloat16,
                        device="cuda")
    pages = torch.randperm(B * width, generator=g).view(B, width).to(torch.int32).cuda()
    shared = prefix // page * page  # whole pages of the common prefix, kept once
    pages[:, :shared // page] = pages[0, :shared // page]
    seqs = [p.tolist() for p in prompts]
    u = torch.rand(steps, B, generator=g).cuda()

    r.alloc_cache(max(map(len, prompts)) + steps)

    def check(logits, rows):
        """Row of every sequence against the runner over the whole sequence so far."""
        for b in range(B):
            want = r.forward(torch.tensor(seqs[b], device="cuda"), 0, use_cache=True)[-1:]
            assert decode_ref.logits_match(logits[rows[b]:rows[b] + 1], want), b

    # prompt step: the sequences' tokens one after the other; the common pages are written by all of
    # them, with the same values
    lens = torch.tensor([len(p) for p in prompts], dtype=torch.int32, device="cuda")
    q_start = F.pad(lens.cumsum(0), (1, 0)).to(torch.int32)
    work = kernels.paged_attention_workspace(int(q_start[-1]), B, shape.heads, shape.kv_heads, shape.head_dim,
                                             width * page, ragged=True, shared=shared)
    x = r.embed.index_select(0, torch.cat(prompts))
    logits = _batch_forward(r, x, pools, pages, lens, q_start, shared, work)
    rows = (q_start[1:] - 1).tolist()
    check(logits, rows)
    logits = logits[rows]
    work = kernels.paged_attention_workspace(B, B, shape.heads, shape.kv_heads, shape.head_dim, width * page,
                                             shared=shared)
    for step in range(steps):
        tok = kernels.sample(logits, u[step], temperature=0.8, top_k=50, top_p=0.9)
        for b, t in enumerate(tok.tolist()):
            assert 0 <= t < shape.vocab
            seqs[b].append(t)
        lens += 1
        logits = _batch_forward(r, r.embed.index_select(0, tok.long()), pools, pages, lens, None, shared, work)
        check(logits, range(B))


def test_generate_samples(kernels):
    """The runner's sampling: temperature 0 is the greedy path's tokens, a seed's numbers give one text,
    eager or from the graph, and each token is what sample draws from the step's logits."""
    shape = Qwen2Shape(layers=2, hidden=512, heads=4, kv_heads=2, intermediate=1024, vocab=2000)
    r = Qwen2Runner.random(shape, seed=4, kernels=kernels)
    ids = torch.randint(0, shape.vocab, (20,), generator=torch.Generator().manual_seed(1)).cuda()
    n = 12
    u = torch.rand(n, generator=torch.Generator().manual_seed(2)).cuda()
    greedy = r.generate(ids, n)
    assert r.generate(ids, n, temperature=0.0, u=u) == greedy
    assert r.generate(ids, n, temperature=0.9, top_k=1, u=u) == greedy
    kw = dict(temperature=1.2, top_k=100, top_p=0.95, min_p=0.001, u=u)
    text = r.generate(ids, n, **kw)
    assert text != greedy and text == r.generate(ids, n, use_graph=False, **kw) == r.generate(ids, n, **kw)
    r.alloc_cache(len(ids) + n)
    logits = r.forward(ids, 0, use_cache=True, last_only=True)
    for i in range(n):
        assert int(kernels.sample(logits, u[i:i + 1], 1.2, 100, 0.95, 0.001)) == text[i]
        if i + 1 < n:
            logits = r.decode(text[i], len(ids) + i)
    assert len(r.generate(ids, n, temperature=1.0)) == n
    with pytest.raises(ValueError):
        r.generate(ids, n, temperature=1.0, u=u[:3])


def test_generate_without_a_token(kernels):
    """Logits that are all NaN leave nothing to draw: -1, which the next step takes as a zero embedding, eager or
    replayed. A temperature below zero or NaN is refused."""
    shape = Qwen2Shape(layers=1, hidden=512, heads=4, kv_heads=2, intermediate=1024, vocab=2000)
    r = Qwen2Runner.random(shape, seed=4, kernels=kernels)
    ids = torch.arange(20).cuda()
    for t in (-0.5, math.nan):
        with pytest.raises(ValueError):
            r.generate(ids, 3, temperature=t)
    r.final_norm.fill_(math.nan)
    for graph in (True, False):
        assert r.generate(ids, 4, use_graph=graph, temperature=0.8, top_k=50, top_p=0.9) == [-1] * 4
