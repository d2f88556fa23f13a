"""Kernels.beam_select and Kernels.paged_reorder against float64 and lists."""
import math

import pytest
import torch

BF16, FP8, E8M0, U8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.uint8
pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ selection
def _want(logits, scores, n):
    """The n largest sums in float64, by value, then beam, then logit (which a float64 sum may swallow), then token; and
    all of the sums."""
    R, beams = scores.shape
    V = logits.shape[1]
    x = logits.cpu().double()
    x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    s = scores.cpu().double()
    s = torch.where(torch.isnan(s), -math.inf, s).clamp(max=torch.finfo(torch.float32).max)
    m = x.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    lse = m + (x - m).exp().sum(1, keepdim=True).log()
    c = s.view(-1, 1) + x - torch.where(lse == -math.inf, 0.0, lse)
    c = torch.where((x == -math.inf) | (s.view(-1, 1) == -math.inf), -math.inf, c).view(R, -1)
    order = torch.sort(x, dim=1, descending=True, stable=True).indices + V * (torch.arange(R * beams) % beams)[:, None]
    order = order.view(R, -1)
    best, at = torch.sort(c.gather(1, order), dim=1, descending=True, stable=True)
    n_ = min(n, c.shape[1])
    best, at = best[:, :n_], order.gather(1, at[:, :n_])
    none = best == -math.inf
    tokens, parents = torch.where(none, -1, at % V), torch.where(none, -1, at // V)
    pad = torch.full((R, n - n_), -1)
    return torch.cat([best, pad - math.inf], 1), torch.cat([tokens, pad], 1), torch.cat([parents, pad], 1), c


def _check(kernels, logits, scores, n, near_ties=False, **kw):
    """Scores to half a step of fp32 and 2^-20 (exponentials in 32 bits: 2^-22 of each weight and their argument's
    rounding, 2^-24 of up to 100 where a weight of e^-100 does not count). Tokens and parents are the exact ones,
    but, with near_ties, where two beams' sums lie closer than that."""
    got = kernels.beam_select(logits, scores, n, **kw)
    torch.cuda.synchronize()
    best, tokens, parents, c = _want(logits, scores, n)
    s, t, p = (x.cpu() for x in got)
    assert s.dtype == torch.float32 and t.dtype == p.dtype == torch.int32
    near = best.abs() * 2.0 ** -24 + 2.0 ** -20
    fin = best > -math.inf
    assert torch.equal(s > -math.inf, fin)
    assert bool(((s.double() - best).abs() <= near)[fin].all())
    same = (t == tokens) & (p == parents)
    V = logits.shape[1]
    for r, k in (~same).nonzero().tolist():
        assert t[r, k] >= 0 and abs(c[r, p[r, k] * V + t[r, k]] - best[r, k]) <= 2.0 ** -20, (r, k)
        others = [j for j in range(best.shape[1]) if j != k and abs(best[r, j] - best[r, k]) <= 2.0 ** -20]
        assert any(parents[r, j] != parents[r, k] for j in others) or k == best.shape[1] - 1
    flat = p.long() * V + t
    for r in range(scores.shape[0]):  # nothing twice
        live = flat[r][fin[r]]
        assert live.unique().numel() == live.numel()
    assert near_ties or bool(same.all())
    return got


def _logits(rows, V, dtype, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, V + pad, generator=g) * 2
    hot = torch.randint(0, V, (rows, 12), generator=g)
    x.scatter_add_(1, hot, torch.rand(rows, 12, generator=g) * 12)
    return x.to(dtype).cuda()[:, :V]


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("R,beams,n,V,pad", [
    (1, 1, 1, 1, 0), (1, 1, 3, 2, 0), (2, 4, 8, 7, 1), (1, 4, 8, 4096, 0), (3, 4, 8, 4097, 3), (1, 4, 8, 152064, 0),
    (5, 3, 6, 32003, 5), (16, 8, 16, 9001, 0), (1, 64, 64, 5000, 7), (2, 33, 64, 20000, 0), (300, 2, 4, 1000, 1),
    (1, 1, 64, 100000, 0), (7, 16, 32, 50257, 1)])
def test_select(kernels, dtype, R, beams, n, V, pad):
    g = torch.Generator().manual_seed(V)
    scores = (-20 - 4 * torch.rand(R, beams, generator=g)).cuda()
    _check(kernels, _logits(R * beams, V, dtype, V + n, pad), scores, n)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_select_equal_logits(kernels, dtype):
    """Ties: within a row, over whole rows, between beams of equal scores."""
    scores = torch.tensor([[-1.0, -1.0, -2.0], [0.0, 0.0, 0.0]], device="cuda")
    for V in (5, 64, 6000, 152064):
        x = torch.zeros(6, V, device="cuda", dtype=dtype)
        _check(kernels, x, scores, 9)
        x[:, ::3] = 1.0
        x[4, V // 2:] = 1.0
        _check(kernels, x, scores, 33)
        _check(kernels, (torch.arange(V, device="cuda") % 7).to(dtype).expand(6, V).contiguous(), scores, 64)


@pytest.mark.parametrize("V", [1000, 152064])
def test_select_orders_that_lengthen_lists(kernels, V):
    """Rows that rise, fall, or hold their largest in one lane's or one part's reach. The first two are each other's
    mirror image (i / V and -(V - 1 - i) / V differ by the same for all i), so their sums tie but for the logits' rounding."""
    scores = torch.full((1, 5), -3.0, device="cuda")
    at = torch.arange(V, device="cuda", dtype=torch.float32)
    x = torch.stack([at / V, -at / V, (at % 4096 < 16).float() + at / V, ((at // 8) % 256 == 3).float() + at / V,
                     (at > V - 200).float() - at / V])
    _check(kernels, x, scores, 64, near_ties=True)
    _check(kernels, x, scores, 10, near_ties=True)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_select_dead_beams_nan_and_infinities(kernels, dtype):
    inf, nan = math.inf, math.nan
    V = 5000
    x = _logits(12, V, dtype, 3)
    x[1] = -inf
    x[2] = nan
    x[3, ::2] = nan
    x[4, 7] = inf
    x[5, 9] = x[5, 4000] = inf
    x[6, 3:] = -inf
    scores = torch.tensor([[-1.0, -1.5, -2.0, -1.0], [-1.0, -2.0, -1.0, nan], [-inf] * 4], device="cuda")
    _check(kernels, x, scores, 20)
    # the step after a prompt: one beam counts
    first = torch.full((3, 4), -inf, device="cuda")
    first[:, 0] = 0.0
    got = _check(kernels, x, first, 8)
    assert bool((got[2][1] <= 0).all())
    _check(kernels, x, torch.full((3, 4), inf, device="cuda"), 8)
    # fewer continuations than asked for
    few = torch.full((4, 30), -inf, device="cuda", dtype=dtype)
    few[0, 3] = few[2, 5] = 0.0
    few[2, 1] = 1.0
    got = _check(kernels, few, torch.tensor([[-1.0, -2.0], [-1.0, -1.0]], device="cuda"), 5)
    assert got[1].tolist() == [[3, -1, -1, -1, -1], [1, 5, -1, -1, -1]]


def test_select_far_scores(kernels):
    """Sums far from the logits' size, where a step of fp32 is wider than what decides."""
    g = torch.Generator().manual_seed(1)
    scores = (-3000 - 1e-3 * torch.rand(4, 8, generator=g)).cuda()
    _check(kernels, _logits(32, 30000, torch.float32, 5), scores, 16)


def test_select_maxima_that_rise(kernels):
    """Rows in parts of several tiles whose maximum rises from tile to tile, a little or by more than fp32 holds; and beams
    that do not count beside them."""
    beams, n, V = 16, 32, 152064
    x = _logits(beams, V, torch.float32, 21)
    at = torch.arange(V, device="cuda", dtype=torch.float32)
    x[0] = at * (60 / V)
    x[1] = -at * (60 / V)
    x[2], x[2, 11000] = -3e38, 3e38
    x[3], x[3, V - 1] = -80.0, 20.0
    x[4], x[4, ::5000] = -math.inf, at[::5000] / 1000
    scores = torch.linspace(-9, -5, beams, device="cuda").view(1, beams)
    _check(kernels, x, scores, n)
    for live in (1, 2, 5):
        some = torch.full_like(scores, -math.inf)
        some[0, 4:4 + live] = scores[0, :live]
        _check(kernels, x, some, n)
        _check(kernels, x[:, :20001], some, n)


@pytest.mark.parametrize("dtype,n", [(BF16, 9), (torch.float32, 32)])
def test_select_many_rows_with_ties(kernels, dtype, n):
    """Enough rows for the widest tiles: rows that are equal throughout, hold a few values, or rise."""
    R, beams, V = 8, 4, 152064
    x = _logits(R * beams, V, dtype, 31)
    at = torch.arange(V, device="cuda")
    x[0:4] = 0.0
    x[4:8] = (at % 7).to(dtype)
    x[8] = (at >= 100000).to(dtype)
    x[9] = at.to(torch.float32).mul(40 / V).to(dtype)
    x[10], x[10, 5] = -3e38, 3e38
    x[11] = math.nan
    scores = torch.linspace(-4, -2, R * beams, device="cuda").view(R, beams)
    scores[0] = -1.0
    _check(kernels, x, scores, n)


@pytest.mark.parametrize("R,beams,n,V", [(2, 2, 64, 32000), (1, 3, 50, 12289), (3, 1, 17, 4097), (1, 64, 1, 152064),
                                         (1, 64, 2, 100001), (4, 5, 63, 8191)])
def test_select_few_and_many_lists(kernels, R, beams, n, V):
    """Fewer lists than continuations asked for, and more of them than threads that join them."""
    scores = torch.linspace(-4, -3, R * beams, device="cuda").view(R, beams)
    _check(kernels, _logits(R * beams, V, BF16, V), scores, n)
    _check(kernels, _logits(R * beams, V, torch.float32, V), scores, n)


def test_select_captured_and_given_buffers(kernels):
    R, beams, n, V = 3, 4, 8, 30001
    x, scores = _logits(R * beams, V, BF16, 1), torch.full((R, beams), -1.0, device="cuda")
    work = kernels.beam_select_workspace(R, beams, V, n)
    out = (torch.zeros(R, n, device="cuda"), torch.zeros(R, n, dtype=torch.int32, device="cuda"),
           torch.zeros(R, n, dtype=torch.int32, device="cuda"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.beam_select(x, scores, n, work=work, out=out)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.beam_select(x, scores, n, work=work, out=out)
    for k in range(4):
        x.copy_(_logits(R * beams, V, BF16, 10 + k))
        scores.copy_(torch.rand(R, beams) * -9)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in out]
        work.fill_(255)
        again = _check(kernels, x, scores, n)
        assert all(torch.equal(a, b) for a, b in zip(kept, again))


# ------------------------------------------------------------------ reordering
def _reorder(table, parents, lens, page, pools, blocks):
    """The new table, and pools (lists of uint8 [layers, n_pages, Hk, rows, bytes] on the CPU, and of scales) changed."""
    R, beams = parents.shape
    out = table.clone()
    for r in range(R):
        base = r * beams
        p = [q if 0 <= q < beams else i for i, q in enumerate(parents[r].tolist())]
        keeper = {}
        for i in sorted(range(beams), key=lambda i: (p[i] != i, i)):
            keeper.setdefault(p[i], i)
        ended = [i for i in range(beams) if i not in p]
        for i in range(beams):
            n = lens[base + p[i]]
            w, part = n // page, n % page
            out[base + i, :w] = table[base + p[i], :w]
            if part == 0:
                continue
            src = table[base + p[i], w]
            if keeper[p[i]] == i:
                out[base + i, w] = src
                continue
            dst = out[base + i, w] = table[base + ended.pop(0), w]
            if not (0 <= src < pools[0].shape[1] and 0 <= dst < pools[0].shape[1]):
                continue
            for x in pools:
                x[:, dst, :, :part] = x[:, src, :, :part]
            for x in blocks:
                x[:, dst, :, :-(-part // 16)] = x[:, src, :, :-(-part // 16)]
    return out


def _beams(R, beams, lens, page, seed):
    """A table whose whole pages a request's beams share, with a last page and one spare entry of their own."""
    g = torch.Generator().manual_seed(seed)
    whole = [n // page for n in lens]
    total = sum(whole) + 2 * R * beams
    order = torch.randperm(total, generator=g).to(torch.int32)
    width = max(whole) + 3
    table = torch.full((R * beams, width), -1, dtype=torch.int32)
    at = 0
    for r, w in enumerate(whole):
        rows = slice(r * beams, (r + 1) * beams)
        table[rows, :w] = order[at:at + w]
        table[rows, w:w + 2] = order[at + w:at + w + 2 * beams].view(beams, 2)
        at += w + 2 * beams
    return table, total


def _pools(layers, total, Hk, page, D, fp8, seed, layered):
    """K and V (and scales) of random bits, strided and between each other in one buffer."""
    g = torch.Generator().manual_seed(seed)
    if fp8:
        x = torch.randint(0, 256, (total, layers, 2, Hk, page + 16, D), generator=g, dtype=U8).cuda()
        s = torch.randint(0, 256, (total, layers, 2, Hk, page // 16 + 1), generator=g, dtype=U8).cuda()
        cut = lambda y, i: y[:, :, i].transpose(0, 1)  # noqa: E731
        pools = [cut(x, i)[..., :page, :].view(FP8) for i in range(2)]
        marks = [cut(s, i)[..., :page // 16].view(E8M0) for i in range(2)]
    else:
        x = torch.randint(-30000, 30000, (layers, 2, total, Hk, page + 16, D), generator=g, dtype=torch.int16).cuda()
        pools, marks = [x[:, i, :, :, :page].view(BF16) for i in range(2)], []
    if not layered:
        pools, marks = [p[0] for p in pools], [m[0] for m in marks]
    return x, pools, marks


def _bits(t, layered):
    t = t if layered else t[None]
    return t.contiguous().view(U8 if t.element_size() == 1 else torch.int16).cpu()


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("R,beams,page,layers,lens", [
    (1, 1, 16, 1, [5]), (1, 4, 16, 1, [0]), (3, 4, 16, 3, [33, 48, 1]), (2, 8, 64, 2, [100, 63]), (2, 5, 48, 1, [47, 95]),
    (1, 64, 16, 2, [30]), (4, 3, 256, 1, [255, 256, 257, 600])])
def test_reorder(kernels, fp8, R, beams, page, layers, lens):
    Hk, D = 3, 64
    layered = layers > 1
    table, total = _beams(R, beams, lens, page, seed=beams)
    buf, pools, marks = _pools(layers, total, Hk, page, D, fp8, R, layered)
    rows = torch.tensor(lens, dtype=torch.int32).repeat_interleave(beams)
    g = torch.Generator().manual_seed(9)
    wide = torch.full((R * beams, table.shape[1] + 2), -9, dtype=torch.int32)
    wide[:, :-2] = table
    pages = wide.cuda()[:, :-2]
    for k in range(7):
        cand = torch.randint(0, beams, (R, 2 * beams), generator=g).to(torch.int32)
        if k == 1:
            cand[:] = 0
        elif k == 2:
            cand[:, :beams] = torch.arange(beams)
        elif k == 3:
            cand[:, :beams] = torch.arange(beams).flip(0)
        elif k == 4:
            cand[:] = beams - 1
        elif k == 5:
            cand[:, 0] = -1
            cand[:, -1 + beams] = beams
        parents = cand[:, :beams]
        was = pages.cpu()
        cpu_pools, cpu_marks = ([_bits(t, layered) for t in ts] for ts in (pools, marks))
        want = _reorder(was, parents, rows.tolist(), page, cpu_pools, cpu_marks)
        other = buf.clone()
        got = kernels.paged_reorder(cand.cuda()[:, :beams], pages, rows.cuda(), *pools, *marks)
        torch.cuda.synchronize()
        assert torch.equal(pages.cpu(), was) and torch.equal(got.cpu(), want)
        for now, then in zip([_bits(t, layered) for t in pools + marks], cpu_pools + cpu_marks):
            assert torch.equal(now, then)
        assert torch.equal(buf[..., page:, :], other[..., page:, :])  # between the heads
        again = kernels.paged_reorder(cand.cuda()[:, :beams], pages, rows.cuda(), *pools, *marks, out=torch.empty_like(got))
        torch.cuda.synchronize()
        assert torch.equal(again, got)
        for now, then in zip([_bits(t, layered) for t in pools + marks], cpu_pools + cpu_marks):
            assert torch.equal(now, then)
        pages = got


def test_reorder_entries_outside_the_pool(kernels):
    table, total = _beams(2, 3, [20, 40], 16, seed=1)
    table[0, 1], table[4, 2] = -1, total
    _, pools, marks = _pools(1, total, 2, 16, 64, True, 3, False)
    lens = torch.tensor([20] * 3 + [40] * 3, dtype=torch.int32)
    parents = torch.tensor([[0, 0, 1], [0, 0, 0]], dtype=torch.int32)
    cpu = [[_bits(t, False) for t in ts] for ts in (pools, marks)]
    want = _reorder(table, parents, lens.tolist(), 16, *cpu)
    got = kernels.paged_reorder(parents.cuda(), table.cuda(), lens.cuda(), *pools, *marks)
    torch.cuda.synchronize()
    assert torch.equal(got.cpu(), want)
    for now, then in zip([_bits(t, False) for t in pools + marks], cpu[0] + cpu[1]):
        assert torch.equal(now, then)
