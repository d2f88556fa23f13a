"""Calls of the paged operators that the documentation allows and that few make."""
import pytest
import torch

import paged_ref as R

BF16 = torch.bfloat16
pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("new", [None, [1, 40, 7]])
def test_counts_past_32_bits(kernels, new):
    """A window or first tokens of more than 32 bits show everything, a prefix of more is all that is shared."""
    Hq, Hk, D = 14, 2, 64
    batch = R.PagedBatch([700, 90, 41], new, Hk, D, 16, seed=1)
    q = (torch.randn(batch.T, Hq * D, generator=torch.Generator().manual_seed(1)) * 2).to(BF16).cuda()

    def attend(b=batch, **kw):
        return kernels.paged_attention(q, b.k, b.v, b.table, b.lens, Hq, q_start=b.q_start, **kw)

    want = attend()
    for n in ((1 << 31) - 1, 1 << 31, (1 << 32) + 16, 1 << 40):
        assert torch.equal(attend(window=n), want)
        assert torch.equal(attend(window=16, sinks=n), attend(window=16, sinks=1 << 20))
    # one sequence shares all of its positions with itself
    one = R.PagedBatch([700], None if new is None else [1], Hk, D, 16, seed=2)
    q = q[:1]
    assert torch.equal(attend(one, shared=(1 << 32) + 16), attend(one, shared=one.table.shape[1] * 16))
