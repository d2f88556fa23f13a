"""Attention over a paged cache in 8 bits where its formats end: probabilities beside values that cancel, scales and queries
near the ends of their ranges, scores that fp32 holds and a factor of them does not, batches of more tiles than workgroups."""
import pytest
import torch

import paged_fp8_ref as F
import paged_ref as R

BF16, U8 = torch.bfloat16, torch.uint8
NAN = float("nan")
pytestmark = pytest.mark.gpu


def _queries(T, Hq, D, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, Hq * D, generator=g) * scale).to(BF16).cuda()


def _attend(kernels, batch, q, Hq, **kw):
    got = kernels.paged_attention_fp8(q, *batch.cache(), batch.table, batch.lens, Hq, q_start=batch.q_start, **kw)
    torch.cuda.synchronize()
    return got


def _fill(batch, name, codes, byte):
    """Codes (broadcast over positions) and one scale byte for every position of the batch, and the values they stand for."""
    values, pool, marks = getattr(batch, name), getattr(batch, name + "8"), getattr(batch, name + "s")
    live = ~torch.isnan(values.float())
    codes = codes.to("cuda").float().expand(values.shape).to(F.FP8)
    bits = pool.view(U8)
    bits.copy_(torch.where(live, codes.view(U8), bits))
    there = live.any(3).unflatten(2, (-1, 16)).any(3)
    marks.view(U8).copy_(torch.where(there, byte, 255).to(U8))
    exact = codes.double() * 2.0 ** (byte - 127)
    assert torch.equal(exact.to(BF16).double(), exact)
    setattr(batch, name, torch.where(live, exact, NAN).to(BF16))


def _check(got, want, v):
    """Half a bf16 step of the result (2^-8 of it), and of the largest value v that a token can see: 2^-16 for probabilities of
    16 bits, 2^-13 for fp32 scores up to a few hundred in the exponent (128 products of 2^-24 each) and fp32 sums, 2^-15 for the
    query's terms below 2^-14 of its largest (off by 2^-22 of 8, times keys of 5, a scale of 0.09 and a quarter of 128 dims)."""
    err = (got.cpu().double().view_as(want) - want).abs()
    bound = want.abs() * 2.0 ** -8 + (2.0 ** -16 + 2.0 ** -13 + 2.0 ** -15) * v
    assert bool((err <= bound).all()), float((err - bound).max())


# (positions, new tokens, shared): tiles whole and split, single tokens and tiles behind a shared prefix
BATCHES = [([70, 0, 300, 65, 1], [70, 0, 44, 1, 1], 0), ([2000, 1111], [130, 1], 0), ([33, 700], None, 0),
           ([300, 257, 256, 280], None, 256), ([700, 65, 64, 70], [3, 1, 2, 6], 64)]


@pytest.mark.parametrize("Hq,Hk,D", [(28, 4, 128), (14, 2, 64), (40, 2, 128)])
@pytest.mark.parametrize("lens,new,shared", BATCHES)
def test_values_that_cancel(kernels, lens, new, shared, Hq, Hk, D):
    """Values of 1 and -1: what is left of them shows the probabilities themselves, which have 16 bits on every path."""
    batch = F.Fp8Batch(lens, new, Hk, D, 16, shared=shared, seed=11)
    g = torch.Generator().manual_seed(12)
    _fill(batch, "v", torch.randint(0, 2, tuple(batch.v.shape), generator=g) * 2 - 1, 127)
    q = _queries(batch.T, Hq, D, 13)
    _check(_attend(kernels, batch, q, Hq, shared=shared), R.attention(batch, q, Hq), 1.0)


@pytest.mark.parametrize("Hq,Hk,D", [(8, 2, 128), (8, 2, 64), (40, 2, 128)])
@pytest.mark.parametrize("lens,new,shared", BATCHES)
def test_large_queries_beside_large_scales(kernels, lens, new, shared, Hq, Hk, D):
    """Queries of 2^21 in a dim where the keys are 0, keys of 448 * 2^119 in one where the queries are: scores are 0, not 0 times a
    factor that passes fp32."""
    batch = F.Fp8Batch(lens, new, Hk, D, 16, shared=shared, seed=14, spread=0)
    codes = torch.zeros(D)
    codes[2] = 448.0
    _fill(batch, "k", codes, 119 + 127)
    q = torch.zeros(batch.T, Hq, D)
    q[:, :, 0] = 2.0 ** 21
    q = q.view(batch.T, -1).to(BF16).cuda()
    want = R.attention(batch, q, Hq)
    _check(_attend(kernels, batch, q, Hq, shared=shared), want, 8.0)


@pytest.mark.parametrize("Hq,Hk,D", [(8, 2, 128), (8, 2, 64), (40, 2, 128)])
@pytest.mark.parametrize("lens,new,shared", BATCHES)
@pytest.mark.parametrize("large,less,e,q0,q1", [(1.0, 0.875, 14, 2.0 ** 8, 1.75 * 2.0 ** -4), (1.0, 0.875, 44, 2.0 ** 8, 1.75 * 2.0 ** -4),
                                                (2.0 ** -8, 2.0 ** -9, 119, 2.0 ** 21, 1.75 * 2.0 ** 8)])
def test_large_scores(kernels, lens, new, shared, large, less, e, q0, q1, Hq, Hk, D):
    """Scores of 0 and finite ones far from it, in the last case where queries and scales together pass fp32: the tokens of the
    largest share the weight (the next ones are 0.22 * 2^10 / 11.3 or more below, e^-19)."""
    batch = F.Fp8Batch(lens, new, Hk, D, 16, shared=shared, seed=15, spread=0)
    codes = torch.zeros(16, D)
    codes[1::3, 1], codes[2::5, 1] = large, less
    codes[:, 2] = 448.0
    _fill(batch, "k", codes.repeat(batch.k.shape[2] // 16, 1), e + 127)
    q = torch.zeros(batch.T, Hq, D)
    q[:, :, 0], q[:, :, 1] = q0, q1
    q = q.view(batch.T, -1).to(BF16).cuda()
    _check(_attend(kernels, batch, q, Hq, shared=shared), R.attention(batch, q, Hq), 8.0)


@pytest.mark.parametrize("Hq,Hk,D", [(8, 2, 128), (8, 2, 64), (40, 2, 128)])
@pytest.mark.parametrize("lens,new,shared", BATCHES)
def test_scales_of_byte_zero(kernels, lens, new, shared, Hq, Hk, D):
    """2^-127, which no append writes and fp32's normal numbers do not reach: for keys, and for values (all with the same
    probability, so that no product is smaller than they are)."""
    batch = F.Fp8Batch(lens, new, Hk, D, 16, shared=shared, seed=16, spread=0)
    g = torch.Generator().manual_seed(17)
    size = tuple(batch.k.shape)
    _fill(batch, "k", torch.randint(2, 8, size, generator=g) * (torch.randint(0, 2, size, generator=g) * 2 - 1), 0)
    q = (torch.randn(batch.T, Hq * D, generator=g) * 2.0 ** 124).to(BF16).cuda()
    _check(_attend(kernels, batch, q, Hq, shared=shared), R.attention(batch, q, Hq), 8.0)
    _fill(batch, "v", torch.randint(2, 8, size, generator=g) * 64, 0)
    q.zero_()
    got, up = _attend(kernels, batch, q, Hq, shared=shared).double(), 2.0 ** 127
    _check(got * up, R.attention(batch, q, Hq) * up, 448.0)


@pytest.mark.parametrize("Hq,Hk,D,lens,new", [
    (32, 16, 64, [300, 310, 200], [300, 250, 200]), (28, 4, 128, [500 + 3 * i for i in range(60)], [1 + i % 30 for i in range(60)]),
    (8, 4, 64, [40 + 7 * i for i in range(70)], [1 + i % 5 for i in range(70)]),
    (16, 8, 128, [40 + 7 * i for i in range(70)], [1 + i % 5 for i in range(70)]),
    (64, 64, 64, [700, 31, 1], [130, 31, 1]), (32, 32, 64, [2500, 1400], [500, 300])])
def test_many_tiles(kernels, Hq, Hk, D, lens, new):
    """Tiles times kv heads from two fifths of the workgroups aimed at to more than they are, of few blocks and of many, of up to
    64 sequences and of more."""
    batch = F.Fp8Batch(lens, new, Hk, D, 16, seed=18, spread=0)
    q = _queries(batch.T, Hq, D, 19)
    v = batch.v.float().nan_to_num(0, 0, 0).abs().amax().item()
    _check(_attend(kernels, batch, q, Hq), R.attention(batch, q, Hq), v)
    kw = dict(window=100, sinks=5)
    _check(_attend(kernels, batch, q, Hq, **kw), R.attention(batch, q, Hq, **kw), v)
