"""ns_sample against its definition in float64: a token per row from temperature, top-k, top-p, min-p
and a given random number."""
import math

import pytest
import torch

BF16 = torch.bfloat16
pytestmark = pytest.mark.gpu


def reference(logits, u, T, k, p, m):
    """(token, margin) of one row in float64: margin is how far, relative to the sums, the draw and
    top-p's end are from where another token would come out."""
    x = logits.detach().cpu().double()
    x = torch.where(torch.isnan(x), -math.inf, x).clamp(max=torch.finfo(torch.float32).max)
    if x.max() == -math.inf:
        return -1, 1.0
    order = torch.argsort(-x, stable=True)
    if not T > 0:
        return int(order[0]), 1.0
    w = torch.exp((x[order] - x[order[0]]) / T)
    w[x[order] == -math.inf] = 0
    n, margin = x.numel(), 1.0
    if 0 < k < n:
        n = k
    if p < 1:
        c = w[:n].cumsum(0)
        before, goal = c - w[:n], p * c[-1]
        keep = max(int((before < goal).sum()), 1)
        gaps = (before[1:] - goal).abs()
        if gaps.numel():
            margin = min(margin, float(gaps.min() / c[-1]))
        n = keep
    n = max(int((w[:n] >= min(m, 1.0)).sum()), 1)
    kept, back = order[:n].sort()
    c = w[:n][back].cumsum(0)
    goal = max(u, 0.0) * c[-1]
    i = min(int((c <= goal).sum()), int((c < c[-1]).sum()))
    margin = min(margin, float((c[:-1] - goal).abs().min() / c[-1]) if n > 1 else 1.0)
    return int(kept[i]), margin


def _settings(B, V, g):
    """One row per combination of settings, cycling."""
    T = [1.0, 0.7, 0.05, 3.0, 100.0, 0.0]
    k = [0, 1, 2, 20, max(V // 3, 1), V, V + 5]
    p = [1.0, 0.9, 0.5, 0.01, 0.0, 0.999]
    m = [0.0, 0.0, 0.05, 0.5, 1.0]

    def pick(v, dtype):
        return torch.tensor([v[i] for i in torch.randint(0, len(v), (B,), generator=g)], dtype=dtype)
    return pick(T, torch.float32), pick(k, torch.int32), pick(p, torch.float32), pick(m, torch.float32)


def _compare(got, x, u, T, k, p, m):
    """Equal tokens wherever the definition's margin is above the weights' rounding: V halves of 2^-42
    of the largest, of a sum of at least the largest."""
    sure = 0
    for r in range(x.shape[0]):
        want, margin = reference(x[r], float(u[r]), float(T[r]), int(k[r]), float(p[r]), float(m[r]))
        if margin > x.shape[1] * 2.0 ** -42:
            sure += 1
            assert int(got[r]) == want, (r, float(u[r]), float(T[r]), int(k[r]), float(p[r]), float(m[r]))
    return sure


# vocabularies of one token and of a partial vector, around a workgroup's vectors (8192) and the list
# (2048), the model's; flat rows, peaked rows, rows of few values (many ties)
@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 63, 1000, 2047, 2049, 8191, 8200, 50257, 152064])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("kind", ["flat", "peaked", "ties"])
def test_sample(kernels, V, dtype, kind):
    B = 96 if V < 10000 else 40
    g = torch.Generator().manual_seed(V)
    x = torch.randn(B, V + 3, generator=g)
    x = {"flat": x * 0.1, "peaked": x * 4, "ties": (x * 2).round()}[kind]
    x[:, ::17] = -math.inf
    x[0] = -math.inf
    x[1] = float("nan")
    x[2, ::2] = float("nan")
    x[3] = 0.0
    x[4] = torch.where(x[4] > 0, 0.0, -0.0)
    x[5] = torch.finfo(dtype).min
    x[6, V // 2] = math.inf
    x = x.to(dtype).cuda()[:, 1:V + 1]  # rows start anywhere
    u = torch.rand(B, generator=g)
    u[7:10] = torch.tensor([0.0, 1 - 2.0 ** -24, 0.5])
    T, k, p, m = _settings(B, V, g)
    got = kernels.sample(x, u.cuda(), T.cuda(), k.cuda(), p.cuda(), m.cuda())
    again = kernels.sample(x, u.cuda(), T.cuda(), k.cuda(), p.cuda(), m.cuda())
    assert torch.equal(got, again)
    sure = _compare(got.cpu(), x.cpu(), u, T, k, p, m)
    assert sure > B // 2
    # scalars are the same settings for all rows
    for i in (10, 11):
        got = kernels.sample(x, u.cuda(), float(T[i]), int(k[i]), float(p[i]), float(m[i]))
        one = [t[i].expand(B) for t in (T, k, p, m)]
        _compare(got.cpu(), x.cpu(), u, *one)


def test_draw_follows_the_weights(kernels):
    """Equal logits: the token is floor(u V); the last kept one for u from 1 on, the first below 0."""
    V = 5000
    u = (torch.arange(V).double() + 0.5) / V
    x = torch.full((V, V), 2.5, dtype=BF16, device="cuda")
    got = kernels.sample(x, u.float().cuda())
    assert torch.equal(got.cpu(), torch.arange(V, dtype=torch.int32))
    # half of the tokens by top-p and by top-k, the first ones by index
    for kw in (dict(top_p=0.5), dict(top_k=V // 2)):
        got = kernels.sample(x, u.float().cuda(), **kw)
        assert torch.equal(got.cpu(), (torch.arange(V) // 2).to(torch.int32))
    odd = torch.tensor([1.0, 7.0, -1.0, float("nan")]).cuda()
    assert kernels.sample(x[:4], odd).tolist() == [V - 1, V - 1, 0, 0]
    # weights 4 : 2 : 1 at indices 2, 0, 1
    x = torch.full((7, 100), -math.inf)
    x[:, 2], x[:, 0], x[:, 1] = math.log(4.0), math.log(2.0), 0.0
    u = (torch.arange(7).float() + 0.5) / 7
    assert kernels.sample(x.cuda(), u.cuda()).tolist() == [0, 0, 1, 2, 2, 2, 2]
    assert kernels.sample(x.cuda(), u.cuda(), top_k=2).tolist() == [0, 0, 2, 2, 2, 2, 2]  # 1 / 3
    assert kernels.sample(x.cuda(), u.cuda(), top_p=0.5).tolist() == [2] * 7
    assert kernels.sample(x.cuda(), u.cuda(), min_p=0.3).tolist() == [0, 0, 2, 2, 2, 2, 2]
    assert kernels.sample(x.cuda(), u.cuda(), temperature=0.0).tolist() == [2] * 7


# top-k around the rules: as many as tiles (297 of 152064, one thread each; 800 of 409600, two), the list
# (2048), and top-p behind a top-k that no list holds; rows whose candidates crowd one bin or overflow it
@pytest.mark.parametrize("V,ks", [(152064, (296, 297, 298, 2047, 2048, 2049, 20000)), (409600, (799, 800, 801, 2048)),
                                  (1 << 20, (50, 2048, 5000))])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_top_k_rules(kernels, V, ks, dtype):
    g = torch.Generator().manual_seed(V)
    for kind in ("spread", "crowded", "few tiles"):
        x = torch.randn(2, V, generator=g) * 2
        if kind == "crowded":
            x = (x * 3).round() / 3
        if kind == "few tiles":
            x[:, 3000:] -= 1e4
        x = x.to(dtype).cuda()
        u = torch.rand(2, generator=g)
        for k in ks:
            for p, m in ((1.0, 0.0), (0.9, 0.0), (0.7, 0.02)):
                got = kernels.sample(x, u.cuda(), 1.5, k, p, m)
                T, p_, m_ = (torch.full((2,), v, dtype=torch.float32) for v in (1.5, p, m))
                _compare(got.cpu(), x.cpu(), u, T, torch.full((2,), k), p_, m_)


# lists around the longest one that is ordered by rank (512), from one token on, with level tokens at the cut
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_list_lengths(kernels, dtype):
    g = torch.Generator().manual_seed(7)
    for V in (5000, 152064):
        x = (torch.randn(2, V, generator=g) * 2).to(dtype)
        u = torch.rand(2, generator=g)
        for k in (2, 3, 4, 5, 63, 64, 65, 255, 256, 257, 510, 511, 512, 513, 514, 1025):
            for p in (1.0, 0.6):
                got = kernels.sample(x.cuda(), u.cuda(), 1.2, k, p)
                T, p_, m_ = (torch.full((2,), v, dtype=torch.float32) for v in (1.2, p, 0.0))
                _compare(got.cpu(), x, u, T, torch.full((2,), k), p_, m_)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_extreme_temperatures_and_logits(kernels, dtype):
    """Temperatures from the least normal number to infinity; logits of the type's lowest and highest."""
    V, B = 3001, 24
    g = torch.Generator().manual_seed(11)
    x = torch.randn(B, V, generator=g)
    top = torch.finfo(dtype).max
    x[1::4] *= 1e30
    x[2::4] = torch.where(x[2::4] > 1, top, -top)
    x[3::4] = torch.where(x[3::4] > 0, x[3::4], torch.tensor(torch.finfo(dtype).min))
    x = x.to(dtype)
    u = torch.rand(B, generator=g)
    for T in (1.2e-38, 1e-30, 1e-3, 1e3, 1e30, math.inf):
        for k, p, m in ((0, 1.0, 0.0), (7, 1.0, 0.0), (0, 0.6, 0.0), (0, 1.0, 0.3), (2500, 0.5, 0.1)):
            got = kernels.sample(x.cuda(), u.cuda(), T, k, p, m)
            T_, p_, m_ = (torch.full((B,), v, dtype=torch.float32) for v in (T, p, m))
            _compare(got.cpu(), x, u, T_, torch.full((B,), k), p_, m_)


@pytest.mark.parametrize("B", [1, 3, 64])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_graph_replays(kernels, B, dtype):
    """Captured calls read logits, numbers and settings at replay, and do not depend on the batch."""
    V = 32003
    g = torch.Generator(device="cuda").manual_seed(B)
    x = (torch.randn(B, V, generator=g, device="cuda") * 3).to(dtype)
    u = torch.rand(B, generator=g, device="cuda")
    p = torch.full((B,), 0.9, device="cuda")
    work = kernels.sample_workspace(B, V, dtype)
    out = torch.zeros(B, dtype=torch.int32, device="cuda")

    def call():
        kernels.sample(x, u, 0.8, 0, p, 0.01, work=work, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for step in range(5):
        x.copy_((torch.randn(B, V, generator=g, device="cuda") * (1 + step)).to(dtype))
        u.copy_(torch.rand(B, generator=g, device="cuda"))
        p.fill_(1.0 - 0.2 * step)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        call()
        assert torch.equal(out, got)
        single = [int(kernels.sample(x[r:r + 1], u[r:r + 1], 0.8, 0, 1.0 - 0.2 * step, 0.01)) for r in range(min(B, 3))]
        assert got[:3].tolist() == single
        _compare(got.cpu(), x.cpu(), u.cpu(), torch.full((B,), 0.8), torch.zeros(B), p.cpu(), torch.full((B,), 0.01))
