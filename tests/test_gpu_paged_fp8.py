"""Attention over a paged cache in 8 bits against float64 over the values that it stands for."""
import pytest
import torch

import paged_fp8_ref as F
import paged_ref as R

BF16 = torch.bfloat16
pytestmark = pytest.mark.gpu

LAYOUTS = [(28, 4, 128), (14, 2, 64), (3, 3, 64), (16, 1, 128), (40, 2, 128), (130, 1, 64)]


def _queries(T, Hq, D, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, Hq * D + 8, generator=g) * scale  # strided rows
    return x.to(BF16).cuda()[:, :Hq * D]


def _check(got, want, batch, scale=1.0, shared=0):
    """Half a bf16 step of the result (2^-8 of it), and of the largest value a token can see: 2^-16 for the
    probabilities' two terms, 2^-14 for fp32 scores up to a few hundred in the exponent (128 products of 2^-24 each) and
    fp32 sums, 2^-14 for the query's terms: values below 2^-14 of the largest are off by 2^-22 of it at most, with 8 the
    largest, keys of 5 and a scale of 0.09 2^-19 each, in not more than a quarter of the dims. In tiles (with q_start, behind a
    shared prefix, more than 16 query heads) probabilities are one bf16 term, each off by 2^-9 of itself, as a sum by 2^-9 of
    the largest value at most; as the errors are independent, the 2-norm over all outputs stays near that of the
    results' rounding, 2^-9 of theirs: within twice that, and 2^-13 of the values besides."""
    v = batch.v.float().nan_to_num(0, 0, 0).abs().amax().item()
    err = (got.cpu().double().view_as(want) - want).abs()
    tiles = batch.q_start is not None or shared > 0 or want.shape[1] // batch.Hk > 16
    bound = want.abs() * 2.0 ** -8 + (2.0 ** -13 + 2.0 ** -14 + (2.0 ** -9 if tiles else 0.0)) * v * scale
    assert bool((err <= bound).all()), float((err - bound).max())
    norm = torch.linalg.vector_norm
    assert norm(err) <= 2.0 ** -8 * norm(want) + 2.0 ** -13 * v * scale * want.numel() ** 0.5


def _attend(kernels, batch, q, Hq, **kw):
    out = torch.full((batch.T, Hq * batch.D), 7.0, dtype=BF16, device="cuda")
    got = kernels.paged_attention_fp8(q, *batch.cache(), batch.table, batch.lens, Hq, q_start=batch.q_start, out=out,
                                      **kw)
    assert got is out
    again = kernels.paged_attention_fp8(q, *batch.cache(), batch.table, batch.lens, Hq, q_start=batch.q_start, **kw)
    torch.cuda.synchronize()
    assert torch.equal(again.view(torch.int16), got.view(torch.int16))
    return got


# lengths of zero and one, around a group (16), a block (32), a page and a workgroup's range (128), many ranges
LENS = [[1], [700], [0, 1, 2, 15, 16, 17, 31, 33], [127, 128, 129, 5, 1000, 0, 2049, 640],
        [3 * i % 200 for i in range(70)]]


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("lens", range(len(LENS)))
@pytest.mark.parametrize("page", [16, 48])
def test_one_token(kernels, Hq, Hk, D, lens, page):
    batch = F.Fp8Batch(LENS[lens], None, Hk, D, page, seed=lens)
    q = _queries(batch.T, Hq, D, lens)
    _check(_attend(kernels, batch, q, Hq), R.attention(batch, q, Hq), batch)


@pytest.mark.parametrize("Hq,Hk,D", [(28, 4, 128), (14, 2, 64), (40, 2, 128)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 3), (100, 4), (128, 200), (5000, 2)])
def test_one_token_window(kernels, Hq, Hk, D, window, sinks):
    batch = F.Fp8Batch([1, 16, 100, 333, 1500, 5001], None, Hk, D, 32, seed=window)
    q = _queries(batch.T, Hq, D, window)
    _check(_attend(kernels, batch, q, Hq, window=window, sinks=sinks), R.attention(batch, q, Hq, window, sinks), batch)


# (positions, new tokens): prompts from 0, chunks behind cached tokens, single tokens, sequences without any
PROMPTS = [([1], [1]), ([100], [100]), ([70, 0, 300, 65, 1], [70, 0, 44, 1, 1]), ([2000, 1111], [130, 1]),
           ([33 + 5 * i for i in range(40)], [i % 7 for i in range(40)])]


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_prompts(kernels, Hq, Hk, D, case):
    lens, new = PROMPTS[case]
    batch = F.Fp8Batch(lens, new, Hk, D, 16 if case % 2 else 48, seed=case)
    q = _queries(batch.T, Hq, D, case)
    _check(_attend(kernels, batch, q, Hq), R.attention(batch, q, Hq), batch)


@pytest.mark.parametrize("Hq,Hk,D", [(28, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 0), (64, 5), (100, 70), (700, 1)])
def test_prompts_window(kernels, Hq, Hk, D, window, sinks):
    batch = F.Fp8Batch([300, 900, 64, 7], [300, 50, 3, 7], Hk, D, 16, seed=sinks)
    q = _queries(batch.T, Hq, D, window)
    _check(_attend(kernels, batch, q, Hq, window=window, sinks=sinks), R.attention(batch, q, Hq, window, sinks), batch)


@pytest.mark.parametrize("Hq,Hk,D", [(28, 4, 128), (14, 2, 64), (40, 2, 128)])
@pytest.mark.parametrize("shared,lens,new", [
    (256, [300, 257, 256, 280], None), (250, [300, 257, 90, 280, 0, 1], None), (64, [700, 65, 64, 70], [3, 1, 2, 6]),
    (100, [100 + 40 * i for i in range(9)], [1 + i % 3 for i in range(9)])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (60, 3)])
def test_shared_prefix(kernels, Hq, Hk, D, shared, lens, new, window, sinks):
    batch = F.Fp8Batch(lens, new, Hk, D, 16, shared=shared, seed=shared)
    q = _queries(batch.T, Hq, D, shared)
    kw = dict(shared=shared // 16 * 16, window=window, sinks=sinks)
    _check(_attend(kernels, batch, q, Hq, **kw), R.attention(batch, q, Hq, window, sinks), batch, shared=shared)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [None, [3, 1, 2]])
def test_scales_from_end_to_end(kernels, D, new):
    """Keys and values far from 1: the scales' range, and scales that differ from block to block."""
    Hq, Hk = 4, 2
    batch = F.Fp8Batch([100, 37, 64], new, Hk, D, 16, spread=0, seed=D)
    for name, by in (("k", -60), ("v", -97)):
        codes, scales = getattr(batch, name + "8"), getattr(batch, name + "s")
        b = scales.view(torch.uint8)
        b.copy_(torch.where(b == 255, 255, b.int() + by).to(torch.uint8))
        values = codes.contiguous().view(torch.uint8).view(F.FP8).float()
        by16 = scales.contiguous().view(torch.uint8).int().sub(127).float().exp2().repeat_interleave(16, 2)[..., None]
        setattr(batch, name, (values * by16).to(BF16))
    q = (_queries(batch.T, Hq, D, 1).double() * 2.0 ** 60).to(BF16)
    _check(_attend(kernels, batch, q, Hq), R.attention(batch, q, Hq), batch)


def test_queries_of_wide_range(kernels):
    """Values of one head that span 2^60: what lies far below the largest has no part in a score of fp32."""
    Hq, Hk, D = 8, 2, 128
    for new in (None, [5, 40, 1]):
        batch = F.Fp8Batch([130, 60, 17], new, Hk, D, 16, spread=0, seed=3)
        g = torch.Generator().manual_seed(5)
        q = (torch.randn(batch.T, Hq * D, generator=g) * torch.exp2(torch.randint(-60, 1, (batch.T, Hq * D), generator=g)
                                                                    .float()) * 8).to(BF16).cuda()
        # the small values in every dim: 128 of 2^-22 * 24 * 5 * 0.09, 2^-14 of a step in the exponent
        _check(_attend(kernels, batch, q, Hq), R.attention(batch, q, Hq), batch, scale=2.0)
