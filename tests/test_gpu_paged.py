"""The operators of a batch over a paged cache against float64: ns_paged_append (bias, rotation and
append) and ns_paged_attention (single tokens, prompts, window and first tokens, shared prefix)."""
import pytest
import torch

import paged_ref as R

BF16 = torch.bfloat16
pytestmark = pytest.mark.gpu

# model layouts (query heads, kv heads, head size) and others: one query head per kv head, one kv head,
# more query heads per kv head than the one-token kernel takes
LAYOUTS = [(28, 4, 128), (14, 2, 64), (12, 2, 128), (3, 3, 64), (16, 1, 128), (40, 2, 128), (130, 1, 64)]


def _queries(T, Hq, D, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, Hq * D + 8, generator=g) * scale  # strided rows
    return x.to(BF16).cuda()[:, :Hq * D]


def _check(got, want, batch, scale=1.0):
    """Half a bf16 step of the result (2^-8 of it), and of the largest value a token can see: 2^-16 for
    the probabilities' two terms, and 2^-14 for fp32 scores up to a few hundred in the exponent (128
    products of 2^-24 each) and fp32 sums."""
    v = batch.v.float().nan_to_num(0, 0, 0).abs().amax().item()
    err = (got.cpu().double().view_as(want) - want).abs()
    bound = want.abs() * 2.0 ** -8 + 2.0 ** -13 * v * scale
    assert bool((err <= bound).all()), float((err - bound).max())


def _attend(kernels, batch, q, Hq, **kw):
    out = torch.full((batch.T, Hq * batch.D), 7.0, dtype=BF16, device="cuda")
    got = kernels.paged_attention(q, batch.k, batch.v, batch.table, batch.lens, Hq, q_start=batch.q_start,
                                  out=out, **kw)
    assert got is out
    again = kernels.paged_attention(q, batch.k, batch.v, batch.table, batch.lens, Hq,
                                    q_start=batch.q_start, **kw)
    torch.cuda.synchronize()
    assert torch.equal(again, got)
    return got


# lengths of zero and one, around a block (16), a page and a workgroup's range (128), many ranges
LENS = [[1], [700], [0, 1, 2, 15, 16, 17, 31, 33], [127, 128, 129, 5, 1000, 0, 2049, 640],
        [3 * i % 200 for i in range(70)]]


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("lens", range(len(LENS)))
@pytest.mark.parametrize("page", [16, 48])
def test_one_token(kernels, Hq, Hk, D, lens, page):
    batch = R.PagedBatch(LENS[lens], None, Hk, D, page, seed=lens)
    q = _queries(batch.T, Hq, D, lens)
    _check(_attend(kernels, batch, q, Hq), R.attention(batch, q, Hq), batch)


@pytest.mark.parametrize("Hq,Hk,D", [(28, 4, 128), (14, 2, 64), (40, 2, 128)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 0), (17, 3), (100, 4), (128, 200), (5000, 2)])
def test_one_token_window(kernels, Hq, Hk, D, window, sinks):
    batch = R.PagedBatch([1, 16, 17, 99, 101, 104, 105, 600, 1300, 0], None, Hk, D, 32, seed=window)
    # positions that no token sees hold NaN, and their whole pages are gone
    for b, n in enumerate(batch.host_lens):
        for j in range(sinks, max(n - window, 0)):
            batch.v[int(batch.cpu_table[b, j // 32]), :, j % 32] = float("nan")
            batch.k[int(batch.cpu_table[b, j // 32]), :, j % 32] = float("nan")
        for p in range(n // 32 + 1):
            if 32 * p >= sinks and 32 * p + 32 <= n - window:
                batch.table[b, p] = -1 if p % 2 else 1 << 20
    q = _queries(batch.T, Hq, D, sinks)
    want = R.attention(batch, q, Hq, window, sinks)
    want = R.attention(batch, q, Hq, window, sinks,
                       hidden=lambda b, j: (j >= sinks) & (j < batch.host_lens[b] - window))
    _check(_attend(kernels, batch, q, Hq, window=window, sinks=sinks), want, batch)


PROMPTS = [([1, 2, 3], [1, 1, 2]), ([17, 300, 64, 65], [17, 100, 0, 65]), ([400, 9, 1000], [400, 3, 19]),
           ([5 + 7 * i for i in range(70)], [i % 4 for i in range(70)])]


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("case", range(len(PROMPTS)))
def test_prompts(kernels, Hq, Hk, D, case):
    batch = R.PagedBatch(*PROMPTS[case], Hk, D, 16 + 16 * (case % 2), seed=case)
    q = _queries(batch.T, Hq, D, case)
    _check(_attend(kernels, batch, q, Hq), R.attention(batch, q, Hq), batch)


@pytest.mark.parametrize("Hq,Hk,D", [(28, 4, 128), (14, 2, 64)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (40, 0), (64, 5), (100, 70), (700, 1)])
def test_prompts_window(kernels, Hq, Hk, D, window, sinks):
    batch = R.PagedBatch([400, 9, 1000, 130], [400, 3, 300, 1], Hk, D, 16, seed=sinks)
    q = _queries(batch.T, Hq, D, window)
    for b, (n, nn) in enumerate(zip(batch.host_lens, batch.new)):  # seen by no token of the sequence
        for j in range(sinks, max(n - nn + 1 - window, 0)):
            for pool in (batch.k, batch.v):
                pool[int(batch.cpu_table[b, j // 16]), :, j % 16] = float("nan")
    want = R.attention(batch, q, Hq, window, sinks, hidden=lambda b, j: (j >= sinks) & (
        j < batch.host_lens[b] - batch.new[b] + 1 - window))
    _check(_attend(kernels, batch, q, Hq, window=window, sinks=sinks), want, batch)


# the shared prefix: shorter and longer than a block, longer than some sequences, with few and many
# rows; and the same call without `shared` gives the same results to fp32 rounding
@pytest.mark.parametrize("Hq,Hk,D", [(28, 4, 128), (14, 2, 64), (40, 2, 128)])
@pytest.mark.parametrize("shared,lens,new", [
    (16, [17, 40, 100], None), (100, [101, 150, 333, 100, 40, 0], None), (900, [901 + i for i in range(37)], None),
    (640, [641, 800, 900], [1, 30, 90]), (70, [71, 500, 75, 10], [1, 200, 5, 3])])
@pytest.mark.parametrize("window,sinks", [(0, 0), (60, 3)])
def test_shared_prefix(kernels, Hq, Hk, D, shared, lens, new, window, sinks):
    batch = R.PagedBatch(lens, new, Hk, D, 16, shared=shared, seed=shared)
    q = _queries(batch.T, Hq, D, shared)
    want = R.attention(batch, q, Hq, window, sinks)
    got = _attend(kernels, batch, q, Hq, shared=shared, window=window, sinks=sinks)
    _check(got, want, batch)
    _check(_attend(kernels, batch, q, Hq, window=window, sinks=sinks), want, batch)


def test_rows_behind_the_last_sequence_and_bad_tables(kernels):
    """Rows of no sequence keep what they hold; table entries outside the pool are left out; a length
    past the table is the table's; more new tokens than positions see nothing."""
    Hq, Hk, D = 8, 2, 128
    batch = R.PagedBatch([50, 40, 3], [10, 40, 3], Hk, D, 16, seed=1)
    T = batch.T + 9
    q = _queries(T, Hq, D, 3)
    out = torch.full((T, Hq * D), 7.0, dtype=BF16, device="cuda")
    for shared in (0, 0):
        kernels.paged_attention(q, batch.k, batch.v, batch.table, batch.lens, Hq, q_start=batch.q_start,
                                out=out, shared=shared)
        assert bool((out[batch.T:] == 7).all())
        _check(out[:batch.T], R.attention(batch, q[:batch.T], Hq), batch)
    for entry in (-1, batch.k.shape[0], -(1 << 31), (1 << 31) - 1):
        table = batch.table.clone()
        table[0, 1] = table[1, 0] = entry
        kernels.paged_attention(q, batch.k, batch.v, table, batch.lens, Hq, q_start=batch.q_start, out=out)
        want = R.attention(batch, q[:batch.T], Hq, hidden=lambda b, j: (
            (j // 16 == 1) & (b == 0)) | ((j // 16 == 0) & (b == 1)))
        _check(out[:batch.T], want, batch)
        assert bool((out[10:26] == 0).all())  # sequence 1's first page holds all they may see
        one = R.PagedBatch([50, 40, 3], None, Hk, D, 16, seed=1)
        got = kernels.paged_attention(q[:3], one.k, one.v, table, one.lens, Hq)
        want = R.attention(one, q[:3], Hq, hidden=lambda b, j: (
            (j // 16 == 1) & (b == 0)) | ((j // 16 == 0) & (b == 1)))
        _check(got, want, one)
    # lengths past the table: its rows only; negative ones: none
    full = R.PagedBatch([64, 64], None, Hk, D, 16, seed=2)
    lens = torch.tensor([1 << 30, -5], dtype=torch.int32, device="cuda")
    got = kernels.paged_attention(q[:2], full.k, full.v, full.table[:, :4], lens, Hq)
    _check(got[:1], R.attention(full, q[:2], Hq)[:1], full)
    assert bool((got[1] == 0).all())
    few = R.PagedBatch([2, 2], [5, 2], Hk, D, 16, seed=2)
    got = kernels.paged_attention(q[:7], few.k, few.v, few.table, few.lens, Hq, q_start=few.q_start)
    assert bool((got[:3] == 0).all())
    few.new, few.T = [2, 2], 4
    _check(got[3:], R.attention(few, q[3:7], Hq), few)


def test_scale_and_large_scores(kernels):
    Hq, Hk, D = 4, 2, 64
    batch = R.PagedBatch([300, 77], [60, 77], Hk, D, 16, seed=5)
    q = _queries(batch.T, Hq, D, 1)
    _check(_attend(kernels, batch, q, Hq, scale=0.37), R.attention(batch, q, Hq, scale=0.37), batch)
    # scores of about 10^4: an fp32 score is off by 10^4 * 2^-22 or so in the exponent
    q = _queries(batch.T, Hq, D, 1, scale=3000.0)
    _check(_attend(kernels, batch, q, Hq), R.attention(batch, q, Hq), batch, scale=64.0)


def test_graph_replays_at_other_lengths(kernels):
    """A captured call reads lengths, tables and q_start at replay."""
    Hq, Hk, D = 28, 4, 128
    lens = [900, 3, 250, 64]
    batch = R.PagedBatch(lens, None, Hk, D, 16, shared=3, seed=9)
    q = _queries(4, Hq, D, 2)
    work = kernels.paged_attention_workspace(4, 4, Hq, Hk, D, batch.table.shape[1] * 16, shared=3)
    out = torch.zeros(4, Hq * D, dtype=BF16, device="cuda")
    now = batch.lens.clone()

    def call():
        kernels.paged_attention(q, batch.k, batch.v, batch.table, now, Hq, shared=3, work=work, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for cut in (1, 2, 1, 3):
        batch.host_lens = [n // cut if n > 3 else n for n in lens]
        now.copy_(torch.tensor(batch.host_lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        _check(got, R.attention(batch, q, Hq), batch)
        call()
        assert torch.equal(out, got)


@pytest.mark.parametrize("Hq,Hk,D,page,bias", [(28, 4, 128, 16, True), (3, 3, 64, 48, False),
                                               (2, 1, 256, 32, True), (5, 1, 16, 16, True)])
@pytest.mark.parametrize("lens,new", [([1, 50, 0, 33], None), ([40, 300000, 2, 16], [40, 7, 5, 0]),
                                      ([5 + i for i in range(70)], [i % 3 for i in range(70)])])
def test_append(kernels, Hq, Hk, D, page, bias, lens, new):
    """q heads, the stored rows, and everything else in the pools as it was."""
    B, H = len(lens), Hq + 2 * Hk
    new_ = [1] * B if new is None else new
    T, pad = sum(new_), 0 if new is None else 4
    g = torch.Generator().manual_seed(D + B)
    width = max(-(-n // page) for n in lens)
    qkv = torch.randn(T + pad, H * D + 8, generator=g).to(BF16).cuda()[:, :H * D]
    b_ = torch.randn(H * D, generator=g).to(BF16).cuda() if bias else None
    inv = (1.0 / 1e6 ** (torch.arange(0, D, 2).float() / D)).cuda()
    n_pages = sum(new_) // page + 3 * B + 2
    # pages of the new tokens only; the others are not in the pool
    table, used = torch.full((B, width), -1, dtype=torch.int32), 0
    table[::2] = 1 << 30
    for b in range(B):
        for j in range(max(lens[b] - new_[b], 0) // page, -(-lens[b] // page)):
            table[b, j] = used
            used += 1
    assert used <= n_pages
    if B == 4:
        table[3, (lens[3] - 1) // page] = n_pages  # this one's token is not stored
    pools = torch.full((2, n_pages, Hk, 2, page, D), 9.0, dtype=BF16, device="cuda")
    k, v = pools[0, :, :, 1], pools[1, :, :, 1]
    start = None if new is None else torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
    out = torch.full((T + pad, Hq * D), 7.0, dtype=BF16, device="cuda")
    kernels.paged_append(qkv, b_, inv, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), k, v, Hq,
                         q_start=start, out=out)
    torch.cuda.synchronize()
    pos = torch.tensor([lens[b] - new_[b] + i for b in range(B) for i in range(new_[b])], device="cuda")
    seq = [b for b in range(B) for i in range(new_[b])]
    x = qkv[:T].double() + (b_.double() if bias else 0)
    x = x.view(T, H, D)
    ang = (pos.double()[:, None] * inv.double())[:, None]
    lo, hi = x[:, :Hq + Hk].chunk(2, -1)
    want = torch.cat([torch.cat([lo * ang.cos() - hi * ang.sin(), hi * ang.cos() + lo * ang.sin()], -1),
                      x[:, Hq + Hk:]], 1)
    # half a bf16 step, and of the pair's magnitude a few fp32 steps (angle, sine, two products)
    mag = x.abs().view(T, H, 2, D // 2).amax(2).repeat(1, 1, 2)
    bound = want.abs() * 2.0 ** -8 + mag * 2.0 ** -19
    assert bool((out[T:] == 7).all())
    assert bool(((out[:T].double().view(T, Hq, D) - want[:, :Hq]).abs() <= bound[:, :Hq]).all())
    keep = torch.full((2, n_pages, Hk, 2, page, D), 9.0, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(keep)
    for t in range(T):
        p = int(pos[t])
        pg = int(table[seq[t], p // page]) if p >= 0 else -1
        if 0 <= pg < n_pages:
            for i in range(2):
                keep[i, pg, :, 1, p % page] = want[t, Hq + i * Hk:Hq + (i + 1) * Hk]
                tol[i, pg, :, 1, p % page] = bound[t, Hq + i * Hk:Hq + (i + 1) * Hk]
    assert bool(((pools.double() - keep).abs() <= tol).all())


def test_shared_prefix_behind_an_empty_slot(kernels):
    """A padded batch: the first slot has no positions and no pages, another is shorter than the prefix."""
    Hq, Hk, D = 28, 4, 128
    batch = R.PagedBatch([0, 300, 90, 260], None, Hk, D, 16, shared=256, seed=4)
    batch.table[0] = -1
    batch.table[2, 6:] = 1 << 30
    q = _queries(batch.T, Hq, D, 6)
    got = _attend(kernels, batch, q, Hq, shared=256)
    _check(got, R.attention(batch, q, Hq), batch)
    assert bool((got[0] == 0).all())


@pytest.mark.parametrize("D", [64, 128])
def test_offsets_past_32_bits(kernels, D):
    """Pages whose offsets pass 2^32 bytes and 2^32 elements, for both operators; nothing is written
    elsewhere."""
    Hq, Hk, page = 4, 1, 16
    n_pages = (1 << 32) // (page * D) + 70
    k, v = (torch.empty(n_pages, Hk, page, D, dtype=BF16, device="cuda") for _ in range(2))
    ids = [n_pages - 1, 3, (1 << 31) // (page * D) + 1, n_pages - 40]  # the low words of some collide
    low = [i % ((1 << 32) // (page * D)) for i in ids if i >= (1 << 32) // (page * D)]
    for pool in (k, v):
        for i in low:
            pool[i] = 9.0
    n = page * len(ids) - 5
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(D)
    qkv = torch.randn(n, (Hq + 2 * Hk) * D, generator=g, device="cuda").to(BF16)
    inv = (1.0 / 1e6 ** (torch.arange(0, D, 2).float() / D)).cuda()
    q = kernels.paged_append(qkv, None, inv, table, lens, k, v, Hq, q_start=start)
    got = kernels.paged_attention(q, k, v, table, lens, Hq, q_start=start)
    one = kernels.paged_attention(q[-1:], k, v, table, lens, Hq)
    torch.cuda.synchronize()
    assert all(bool((pool[i] == 9).all()) for pool in (k, v) for i in low)
    kk, vv = (pool[torch.tensor(ids, device="cuda")][:, 0].reshape(-1, D)[:n].double() for pool in (k, v))
    assert torch.equal(vv, qkv[:, (Hq + Hk) * D:].double())
    s = (q.double().view(n, Hq, D).transpose(0, 1).reshape(-1, D) @ kk.t()).view(Hq, n, n) / D ** 0.5
    s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), float("-inf"))
    want = (torch.softmax(s, -1).view(-1, n) @ vv).view(Hq, n, D).transpose(0, 1)
    bound = want.abs() * 2.0 ** -8 + 2.0 ** -13 * vv.abs().amax()
    assert bool(((got.double().view(n, Hq, D) - want).abs() <= bound).all())
    assert bool(((one.double().view(Hq, D) - want[-1]).abs() <= bound[-1]).all())


@pytest.mark.parametrize("n,ragged", [(700001, False), (300007, True)])
def test_long_cache(kernels, n, ragged):
    """Far positions: keys planted at the start, the middle and the end decide the result."""
    Hq, Hk, D, page = 7, 1, 128, 64
    g = torch.Generator(device="cuda").manual_seed(n)
    count = -(-n // page)
    k, v = (torch.randn(count, Hk, page, D, generator=g, device="cuda").to(BF16) for _ in range(2))
    k *= 0.05
    table = torch.randperm(count, generator=g, device="cuda").to(torch.int32)[None]
    T = 5 if ragged else 1
    q = torch.randn(T, Hq * D, generator=g, device="cuda").to(BF16)
    q[:, ::D] = 16.0
    for j in (5, n // 2, n - T - 1, n - 2):
        k[int(table[0, j // page]), 0, j % page, 0] = 18.0
    start = torch.tensor([0, T], dtype=torch.int32, device="cuda") if ragged else None
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    got = kernels.paged_attention(q, k, v, table, lens, Hq, q_start=start).double().view(T, Hq, D)
    kk, vv = (pool[table[0].long(), 0].reshape(-1, D)[:n].double() for pool in (k, v))
    for t in range(T):
        s = q[t].double().view(Hq, D) @ kk[:n - T + t + 1].t() / D ** 0.5
        want = torch.softmax(s, -1) @ vv[:n - T + t + 1]
        err = (got[t] - want).abs()
        assert bool((err <= want.abs() * 2.0 ** -8 + 2.0 ** -13 * vv.abs().amax()).all())


def test_many_sequences(kernels):
    """A batch of a thousand: its items are found over many steps, single tokens and drafts."""
    Hq, Hk, D = 4, 2, 64
    lens = [(37 * i) % 90 for i in range(1000)]
    for new in (None, [min(i % 5, n) for i, n in enumerate(lens)]):
        batch = R.PagedBatch(lens, new, Hk, D, 16, seed=8)
        q = _queries(batch.T, Hq, D, 8)
        _check(_attend(kernels, batch, q, Hq), R.attention(batch, q, Hq), batch)


def test_two_streams(kernels):
    """Calls with workspaces of their own at once on two streams, tensors made on a third."""
    Hq, Hk, D = 28, 4, 128
    batch = R.PagedBatch([3000, 17, 900], None, Hk, D, 16, seed=3)
    q = _queries(batch.T, Hq, D, 1)
    want = _attend(kernels, batch, q, Hq)
    x = torch.randn(3, 50000, generator=torch.Generator().manual_seed(1)).cuda()
    u = torch.rand(3, generator=torch.Generator().manual_seed(2)).cuda()
    tok = kernels.sample(x, u, 0.9, 0, 0.9)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for i in range(6):
        with torch.cuda.stream(streams[i % 2]):
            outs.append((kernels.paged_attention(q, batch.k, batch.v, batch.table, batch.lens, Hq),
                         kernels.sample(x, u, 0.9, 0, 0.9)))
    torch.cuda.synchronize()
    for a, t in outs:
        assert torch.equal(a, want) and torch.equal(t, tok)
