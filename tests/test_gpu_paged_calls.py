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


@pytest.mark.parametrize("layout", ["pages", "heads", "layers"])
def test_pools_cut_from_one_buffer(kernels, layout):
    """Keys and values beside each other per page or per head, or of one layer of a pool of all layers."""
    Hq, Hk, D, page = 14, 2, 64, 16
    batch = R.PagedBatch([70, 33, 5], [3, 33, 1], Hk, D, page, seed=1)
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(batch.T, (Hq + 2 * Hk) * D, generator=g).to(BF16).cuda()
    inv = (1.0 / 1e6 ** (torch.arange(0, D, 2).float() / D)).cuda()
    n = batch.k.shape[0]
    if layout == "pages":
        buf = torch.full((n, 2, Hk, page, D), 9.0, dtype=BF16, device="cuda")
        k, v = buf[:, 0], buf[:, 1]
    elif layout == "heads":
        buf = torch.full((Hk, 2, n, page, D), 9.0, dtype=BF16, device="cuda")
        k, v = (buf[:, i].transpose(0, 1) for i in (0, 1))
    else:
        buf = torch.full((n, 3, 2, Hk, page, D), 9.0, dtype=BF16, device="cuda")
        k, v = buf[:, 1, 0], buf[:, 1, 1]

    def run(k, v):
        q = kernels.paged_append(qkv, None, inv, batch.table, batch.lens, k, v, Hq, q_start=batch.q_start)
        return kernels.paged_attention(q, k, v, batch.table, batch.lens, Hq, q_start=batch.q_start)

    pools = [batch.k.contiguous(), batch.v.contiguous()]
    k.copy_(pools[0])
    v.copy_(pools[1])
    others = buf[:, [0, 2]].clone() if layout == "layers" else None
    want = run(*pools)
    got = run(k, v)
    torch.cuda.synchronize()
    bits = torch.int16  # (the pools' unused rows are NaN)
    assert torch.equal(got, want)
    assert torch.equal(k.contiguous().view(bits), pools[0].view(bits))
    assert torch.equal(v.contiguous().view(bits), pools[1].view(bits))
    if others is not None:
        assert torch.equal(buf[:, [0, 2]], others)


@pytest.mark.parametrize("Hq,Hk,D,shared,window,sinks", [(28, 4, 128, 0, 0, 0), (14, 2, 64, 0, 50, 3), (28, 4, 128, 64, 0, 0),
                                                         (14, 2, 64, 64, 40, 2)])
def test_a_captured_step_of_any_batch(kernels, Hq, Hk, D, shared, window, sinks):
    """One captured step of append and attention with q_start, replayed for other lengths, other numbers of tokens per
    sequence, sequences without any and padded rows; eager work between the replays."""
    page, B, T, width = 16, 4, 64, 30
    g = torch.Generator().manual_seed(D + shared)
    n_pages = B * width
    order = torch.randperm(n_pages, generator=g).view(B, width).to(torch.int32)
    order[:, :shared // page] = order[0, :shared // page]
    table = order.cuda()
    # (the shared rows are written once; every sequence's own follow)
    k, v = (torch.randn(n_pages, Hk, page, D, generator=g).to(BF16).cuda() for _ in range(2))
    qkv = torch.zeros(T, (Hq + 2 * Hk) * D, dtype=BF16, device="cuda")
    inv = (1.0 / 1e6 ** (torch.arange(0, D, 2).float() / D)).cuda()
    lens, start = torch.ones(B, dtype=torch.int32, device="cuda"), torch.arange(B + 1, dtype=torch.int32, device="cuda")
    q, out = (torch.zeros(T, Hq * D, dtype=BF16, device="cuda") for _ in range(2))
    work = kernels.paged_attention_workspace(T, B, Hq, Hk, D, width * page, ragged=True, shared=shared)

    def step(q, out, work):
        kernels.paged_append(qkv, None, inv, table, lens, k, v, Hq, q_start=start, out=q)
        kernels.paged_attention(q, k, v, table, lens, Hq, q_start=start, shared=shared, window=window, sinks=sinks,
                                work=work, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(q, out, work)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(q, out, work)
    for new, total in (([1, 1, 1, 1], [100, 470, 65, 300]), ([40, 0, 3, 1], [480, 0, 70, 90]), ([0, 0, 64, 0], [90, 80, 130, 65]),
                       ([1, 1, 1, 1], [480, 480, 480, 480]), ([16, 16, 16, 16], [80, 300, 81, 479]), ([0, 0, 0, 0], [5, 6, 7, 8])):
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(BF16))
        lens.copy_(torch.tensor(total, dtype=torch.int32))
        start.copy_(torch.tensor([0] + new).cumsum(0).to(torch.int32))
        q.fill_(7.0)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        rows = sum(new)
        assert bool((out[rows:] == 7).all()) and bool((q[rows:] == 7).all())
        again, mine = torch.full_like(out, 7.0), torch.full_like(q, 7.0)
        step(mine, again, None)
        assert torch.equal(again, out) and torch.equal(mine, q)
        batch = R.PagedBatch([1], None, Hk, D, page)  # (the reference's view of these pools)
        batch.host_lens, batch.new, batch.T = total, new, rows
        batch.k, batch.v, batch.cpu_table = k, v, order
        if rows:
            want = R.attention(batch, q[:rows], Hq, window, sinks)
            err = (out[:rows].cpu().double().view_as(want) - want).abs()
            assert bool((err <= want.abs() * 2.0 ** -8 + 2.0 ** -13 * 8.0).all())
