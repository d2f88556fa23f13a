"""Attention over a paged cache in bf16 with finite scores far from 0: no NaN, and the tokens of the largest share the weight."""
import pytest
import torch

import paged_ref as R

BF16 = torch.bfloat16
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hk,D", [(8, 2, 128), (8, 2, 64), (40, 2, 128)])
@pytest.mark.parametrize("lens,new,shared", [([70, 0, 300, 65, 1], [70, 0, 44, 1, 1], 0), ([2000, 1111], [130, 1], 0),
                                             ([33, 700], None, 0), ([300, 257, 256, 280], None, 256),
                                             ([700, 65, 64, 70], [3, 1, 2, 6], 64)])
@pytest.mark.parametrize("by", [10, 40, 110])
def test_large_scores(kernels, lens, new, shared, by, Hq, Hk, D):
    batch = R.PagedBatch(lens, new, Hk, D, 16, shared=shared, seed=by)
    live = ~torch.isnan(batch.k)
    rows = torch.zeros(16, D)
    rows[1::3, 1], rows[2::5, 1] = 2.0 ** by, 0.875 * 2.0 ** by
    batch.k.copy_(torch.where(live, rows.to(BF16).cuda().expand(batch.k.shape), batch.k))
    q = torch.zeros(batch.T, Hq, D)
    q[:, :, 1] = 1.75
    q = q.view(batch.T, -1).to(BF16).cuda()
    got = kernels.paged_attention(q, batch.k, batch.v, batch.table, batch.lens, Hq, q_start=batch.q_start, shared=shared)
    torch.cuda.synchronize()
    want = R.attention(batch, q, Hq)
    # half a bf16 step; equal weights of the largest and e^-19 of the next ones: 2^-16 for probabilities, 2^-20 for the sums
    err = (got.cpu().double().view_as(want) - want).abs()
    assert bool((err <= want.abs() * 2.0 ** -8 + 2.0 ** -15 * 8).all()), float(err.max())
