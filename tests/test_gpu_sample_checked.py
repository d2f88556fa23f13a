"""ns_sample against its definition where test_gpu_sample.py leaves open how many rows were compared: each test counts
the rows whose token the weights' rounding cannot change, and wants nearly all of them. A draw or a cut falls within
e = V 2^-42 of one of n borders with a chance of about 2 e n: at V = 2^20 and n = 20000 one in a hundred."""
import math

import pytest
import torch

import test_gpu_sample as S

BF16 = torch.bfloat16
pytestmark = pytest.mark.gpu


def _run(kernels, x, u, T, k, p, m):
    """Rows compared of one call with scalar settings."""
    B = x.shape[0]
    got = kernels.sample(x.cuda(), u.cuda(), T, k, p, m)
    T_, p_, m_ = (torch.full((B,), v, dtype=torch.float32) for v in (T, p, m))
    return S._compare(got.cpu(), x, u, T_, torch.full((B,), k), p_, m_)


@pytest.mark.parametrize("V,ks", [(152064, (296, 297, 298, 2047, 2048, 2049, 20000)), (409600, (799, 800, 801, 2048)),
                                  (1 << 20, (50, 2048, 5000))])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("kind", ["spread", "crowded", "few tiles"])
def test_top_k_rules(kernels, V, ks, dtype, kind):
    g = torch.Generator().manual_seed(V + 1)
    x = torch.randn(4, V, generator=g) * 2
    if kind == "crowded":
        x = (x * 3).round() / 3
    if kind == "few tiles":
        x[:, 3000:] -= 1e4
    x = x.to(dtype)
    sure = rows = 0
    for k in ks:
        for p, m in ((1.0, 0.0), (0.9, 0.0), (0.7, 0.02)):
            sure += _run(kernels, x, torch.rand(4, generator=g), 1.5, k, p, m)
            rows += 4
    # (a minimum of 0.02 and a crowded row leave level weights, whose borders no rounding moves past each other)
    assert sure >= 0.9 * rows, (sure, rows)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_list_lengths(kernels, dtype):
    g = torch.Generator().manual_seed(17)
    sure = rows = 0
    for V in (5000, 152064):
        x = (torch.randn(3, V, generator=g) * 2).to(dtype)
        for k in (2, 3, 4, 5, 63, 64, 65, 255, 256, 257, 510, 511, 512, 513, 514, 1025):
            for p in (1.0, 0.6):
                sure += _run(kernels, x, torch.rand(3, generator=g), 1.2, k, p, 0.0)
                rows += 3
    assert sure >= 0.95 * rows, (sure, rows)


@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_extreme_temperatures(kernels, dtype):
    g = torch.Generator().manual_seed(19)
    x = (torch.randn(24, 3001, generator=g) * 3).to(dtype)
    sure = rows = 0
    for T in (1.2e-38, 1e-30, 1e-3, 1e3, 1e30, math.inf):
        for k, p, m in ((0, 1.0, 0.0), (7, 1.0, 0.0), (0, 0.6, 0.0), (0, 1.0, 0.3), (2500, 0.5, 0.1)):
            sure += _run(kernels, x, torch.rand(24, generator=g), T, k, p, m)
            rows += 24
    assert sure >= 0.9 * rows, (sure, rows)


# rows whose cut lies in a bin of more than the list's 2048 tokens, which one workgroup cuts alone: high temperatures
# over large vocabularies, few distinct values
@pytest.mark.parametrize("V,T", [(152064, 20.0), (1 << 20, 4.0), (40000, 1e6)])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
@pytest.mark.parametrize("kind", ["normal", "few values"])
def test_crowded_bins(kernels, V, T, dtype, kind):
    g = torch.Generator().manual_seed(V)
    x = torch.randn(3, V, generator=g) * 2
    x = (x.round() if kind == "few values" else x).to(dtype)
    sure = rows = 0
    for k, p, m in ((0, 0.9, 0.0), (0, 0.3, 0.0), (V // 2, 1.0, 0.0), (V // 3, 0.5, 0.0), (V // 2, 0.9, 0.5)):
        sure += _run(kernels, x, torch.rand(3, generator=g), T, k, p, m)
        rows += 3
    # (2 e n is a half at 2^20 tokens of about equal weight)
    assert sure >= (0.25 if V == 1 << 20 else 0.8) * rows, (sure, rows)


@pytest.mark.parametrize("B", [1, 64])
@pytest.mark.parametrize("dtype", [BF16, torch.float32])
def test_graph_replays(kernels, B, dtype):
    V = 32003
    g = torch.Generator(device="cuda").manual_seed(B)
    x = torch.zeros(B, V, dtype=dtype, device="cuda")
    u, p = torch.zeros(B, device="cuda"), torch.ones(B, device="cuda")
    k = torch.zeros(B, dtype=torch.int32, device="cuda")
    work = kernels.sample_workspace(B, V, dtype)
    out = torch.zeros(B, dtype=torch.int32, device="cuda")

    def call():
        kernels.sample(x, u, 0.8, k, p, 0.01, work=work, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    sure = rows = 0
    for step in range(4):
        x.copy_((torch.randn(B, V, generator=g, device="cuda") * (1 + step)).to(dtype))
        u.copy_(torch.rand(B, generator=g, device="cuda"))
        p.fill_(1.0 - 0.2 * step)
        k.fill_((0, 20, 5000, 700)[step])
        graph.replay()
        torch.cuda.synchronize()
        sure += S._compare(out.cpu(), x.cpu(), u.cpu(), torch.full((B,), 0.8), k.cpu(), p.cpu(), torch.full((B,), 0.01))
        rows += B
    assert sure >= 0.75 * rows, (sure, rows)
