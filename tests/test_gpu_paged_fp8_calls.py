"""Calls of the 8-bit cache's operators beside the plain ones: NaN in what a token sees and in what none sees, padded
batches, far pages, captured steps, streams, pools cut from one buffer."""
import math

import pytest
import torch

import paged_fp8_ref as F
import paged_ref as R
from paged_fp8_ref import E8M0, FP8

BF16, U8 = torch.bfloat16, torch.uint8
NAN = float("nan")
pytestmark = pytest.mark.gpu

LAYOUTS = [(28, 4, 128), (14, 2, 64), (40, 2, 128)]
# (lens, new, shared): single tokens of one range and of many, tiles of one range and of many, behind a shared prefix
BATCHES = {
    "one": ([5, 40, 700, 3000, 0, 64], None, 0),
    "one long": ([9000], None, 0),
    "tiles": ([60, 17], [60, 3], 0),
    "tiles split": ([1000, 40], [300, 40], 0),
    "one shared": ([700, 130, 90, 101], None, 96),
    "tiles shared": ([641, 900, 640], [1, 90, 4], 640),
}


def _queries(T, Hq, D, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, Hq * D, generator=g) * 2).to(BF16).cuda()


def _attend(kernels, batch, q, Hq, **kw):
    got = kernels.paged_attention_fp8(q, *batch.cache(), batch.table, batch.lens, Hq, q_start=batch.q_start, **kw)
    torch.cuda.synchronize()
    return got


def _near(got, want, v=8.0 * 16):
    """Where the reference is a number: half a bf16 step of it, 2^-9 of the largest value (spread 4: up to 2^4 * 5)
    for probabilities in one bf16 term, 2^-12 for scores and sums. NaN where the reference has it."""
    got = got.cpu().double().view_as(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    fin = ~torch.isnan(want)
    assert bool(((got - want).abs() <= want.abs() * 2.0 ** -8 + (2.0 ** -9 + 2.0 ** -12) * v)[fin].all())


def _set(batch, name, b, j, value, dim=slice(None)):
    """A code in both the 8-bit pool and the values that it stands for."""
    page, row = int(batch.cpu_table[b, j // batch.page]), j % batch.page
    getattr(batch, name + "8").view(U8)[page, :, row, dim] = torch.tensor([value], device="cuda").to(FP8).view(U8)
    getattr(batch, name)[page, :, row, dim] = NAN if math.isnan(value) else 0.0


def _with_nan(batch, q, Hq, **kw):
    """The reference with NaN keys: NaN for every token that sees one."""
    want = R.attention(batch, q, Hq, **kw)
    k = {}
    for t, b, p in batch.rows():
        if b not in k:
            k[b] = torch.isnan(batch.gather(batch.k, b, max(batch.host_lens[b], 1))).any(2)  # [Hk, n]
        j = torch.arange(k[b].shape[1])
        see = (j <= p) & ((j > p - kw["window"]) | (j < kw["sinks"]) if kw.get("window") else True)
        bad = (k[b] & see).any(1).repeat_interleave(Hq // batch.Hk)
        want[t] = torch.where(bad[:, None], NAN, want[t])
    return want


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("name", BATCHES)
def test_nan_queries_and_keys(kernels, name, Hq, Hk, D):
    lens, new, shared = BATCHES[name]
    batch = F.Fp8Batch(lens, new, Hk, D, 16, shared=shared, seed=7)
    q = _queries(batch.T, Hq, D, 1)
    bad = q.clone()
    bad[0, 3] = NAN
    bad[-1, (Hq - 1) * D + D - 1] = float("inf")  # counts as NaN
    want = R.attention(batch, q, Hq)
    want[0, 0] = want[-1, Hq - 1] = NAN
    last = [b for b, n in enumerate(batch.host_lens) if n > 0 and batch.new[b] > 0]
    if batch.host_lens[-1] <= 0:  # a row that sees nothing stays zero
        want[-1, Hq - 1] = 0.0
    _near(_attend(kernels, batch, bad, Hq, shared=shared), want)
    b = last[-1]
    _set(batch, "k", b, batch.host_lens[b] - 1, NAN, dim=D - 1)
    _set(batch, "k", b, 0, NAN, dim=0)
    _near(_attend(kernels, batch, q, Hq, shared=shared), _with_nan(batch, q, Hq))


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("window,sinks", [(20, 0), (40, 3)])
def test_nan_where_no_token_sees(kernels, name, window, sinks, Hq, Hk, D):
    """Codes of NaN and scales of any byte (255 among them) in positions below every window: no effect."""
    lens, new, shared = BATCHES[name]
    batch = F.Fp8Batch(lens, new, Hk, D, 16, shared=shared, seed=8)
    q = _queries(batch.T, Hq, D, 2)
    kw = dict(window=window, sinks=sinks)
    clean = _attend(kernels, batch, q, Hq, shared=shared, **kw)
    _near(clean, R.attention(batch, q, Hq, **kw))
    seen = {}
    for t, b, p in batch.rows():
        for j in range(max(p + 1, 0)):
            if j > p - window or j < sinks:
                seen.setdefault((int(batch.cpu_table[b, j // 16]), j % 16), True)
    blocks = {pg for pg, _ in seen}
    for b, n in enumerate(batch.host_lens):
        for j in range(max(n, 0)):
            pg = int(batch.cpu_table[b, j // 16])
            if (pg, j % 16) not in seen:
                for pool in (batch.k8, batch.v8):
                    pool.view(U8)[pg, :, j % 16] = 0x7f
            if pg not in blocks and j % 16 == 0:
                batch.ks.view(U8)[pg] = 255
                batch.vs.view(U8)[pg] = 255 if j % 32 else 3
    again = _attend(kernels, batch, q, Hq, shared=shared, **kw)
    assert torch.equal(again.view(torch.int16), clean.view(torch.int16))


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("name", BATCHES)
def test_nan_values(kernels, name, Hq, Hk, D):
    """A NaN code in a value that tokens see: NaN in that dim of theirs alone."""
    lens, new, shared = BATCHES[name]
    batch = F.Fp8Batch(lens, new, Hk, D, 16, shared=shared, seed=9)
    q = _queries(batch.T, Hq, D, 3)
    want = R.attention(batch, q, Hq)
    # the first new token's, which all new ones of the sequence see, and no other sequence
    b, j = [(i, n - batch.new[i]) for i, n in enumerate(batch.host_lens) if n - batch.new[i] >= shared and batch.new[i] > 0 and n > 0][-1]
    _set(batch, "v", b, j, NAN, dim=5)
    got = _attend(kernels, batch, q, Hq, shared=shared).cpu().double().view_as(want)
    row = sum(batch.new[:b])
    rows = slice(row, row + batch.new[b])
    assert bool(torch.isnan(got[rows, :, 5]).all())
    got[rows, :, 5] = want[rows, :, 5]
    _near(got, want)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("new", [None, [3, 1, 2, 4]])
def test_rows_of_no_sequence_and_bad_tables(kernels, D, new):
    """Entries outside the pool are left out; rows in front of and behind the batch's keep what they hold."""
    Hq, Hk = 8, 2
    batch = F.Fp8Batch([100, 37, 0 if new is None else 4, 64], new, Hk, D, 16, seed=D)
    batch.table[0, 2] = -1
    batch.table[1, 0] = 1 << 30
    batch.table[3, 3] = batch.k8.shape[0]
    gone = {0: (32, 48), 1: (0, 16), 3: (48, 64)}

    def hidden(b, j):
        lo, hi = gone.get(b, (0, 0))
        return (j >= lo) & (j < hi)

    q = _queries(batch.T, Hq, D, 4)
    want = R.attention(batch, q, Hq, hidden=hidden)
    if new is None:
        _near(_attend(kernels, batch, q, Hq), want)
        return
    q = torch.cat([q[:2], q, q[:3]])
    out = torch.full_like(q, 7.0)
    kernels.paged_attention_fp8(q, *batch.cache(), batch.table, batch.lens, Hq, q_start=batch.q_start + 2, out=out)
    torch.cuda.synchronize()
    assert bool((out[:2] == 7).all()) and bool((out[-3:] == 7).all())
    _near(out[2:-3], want)


@pytest.mark.parametrize("D", [64, 128])
def test_offsets_past_32_bits(kernels, D):
    """Pages whose offsets pass 2^32 bytes, and scales of theirs; nothing is written elsewhere."""
    Hq, Hk, page = 4, 1, 16
    n_pages = (1 << 32) // (page * D) + 70
    k, v = (torch.empty(n_pages, Hk, page, D, dtype=U8, device="cuda") for _ in range(2))
    # (a page's scale lies a page apart too, in a buffer of its own)
    marks = torch.empty(2, n_pages, page * D // 8, dtype=U8, device="cuda")
    ks, vs = (marks[i][:, None, :1].view(E8M0) for i in range(2))
    ids = [n_pages - 1, 3, (1 << 31) // (page * D) + 1, n_pages - 40]  # the low words of some collide
    low = [i % ((1 << 32) // (page * D)) for i in ids if i >= (1 << 32) // (page * D)]
    for pool in (k, v):
        for i in low:
            pool[i] = 9
    n = page * len(ids) - 5
    table = torch.tensor([ids], dtype=torch.int32, device="cuda")
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    start = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(D)
    qkv = torch.randn(n, (Hq + 2 * Hk) * D, generator=g, device="cuda").to(BF16)
    inv = (1.0 / 1e6 ** (torch.arange(0, D, 2).float() / D)).cuda()
    pools = (k.view(FP8), v.view(FP8), ks, vs)
    q = kernels.paged_append_fp8(qkv, None, inv, table, lens, *pools, Hq, q_start=start)
    got = kernels.paged_attention_fp8(q, *pools, table, lens, Hq, q_start=start)
    one = kernels.paged_attention_fp8(q[-1:], *pools, table, lens, Hq)
    torch.cuda.synchronize()
    assert all(bool((pool[i] == 9).all()) for pool in (k, v) for i in low)
    at = torch.tensor(ids, device="cuda")
    kk, vv = ((c[at].view(FP8).float()[:, 0] * s[at].view(E8M0).float()[:, 0, :, None]).reshape(-1, D)[:n].double()
              for c, s in ((k, ks.view(U8)), (v, vs.view(U8))))
    exact = qkv[:, (Hq + Hk) * D:].double()
    assert bool(((vv - exact).abs() <= exact.abs() * 2.0 ** -4 + 2.0 ** -10 * 8 / 224).all())
    s = (q.double().view(n, Hq, D).transpose(0, 1).reshape(-1, D) @ kk.t()).view(Hq, n, n) / D ** 0.5
    s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool, device="cuda").tril(), float("-inf"))
    want = (torch.softmax(s, -1).view(-1, n) @ vv).view(Hq, n, D).transpose(0, 1)
    bound = want.abs() * 2.0 ** -8 + (2.0 ** -9 + 2.0 ** -12) * vv.abs().amax()
    assert bool(((got.double().view(n, Hq, D) - want).abs() <= bound).all())
    assert bool(((one.double().view(Hq, D) - want[-1]).abs() <= bound[-1]).all())


def _layers(layout, n_pages, Hk, page, D):
    """K, V and their scales cut from one buffer."""
    code, mark = page * D, page // 16
    if layout == "pages":  # a record per page: K, V, then their scales, padded to 16 bytes
        record = 2 * Hk * code + -(-2 * Hk * mark // 16) * 16
        buf = torch.full((n_pages, record), 0x7f, dtype=U8, device="cuda")
        pools = [buf[:, i * Hk * code:(i + 1) * Hk * code].view(n_pages, Hk, page, D) for i in range(2)]
        marks = [buf[:, 2 * Hk * code + i * Hk * mark:2 * Hk * code + (i + 1) * Hk * mark].view(n_pages, Hk, mark)
                 for i in range(2)]
    elif layout == "heads":  # K and V of a head beside each other
        buf = torch.full((n_pages, Hk, 2, page, D), 0x7f, dtype=U8, device="cuda")
        pools = [buf[:, :, i] for i in range(2)]
        both = torch.full((Hk, n_pages, 2, mark), 255, dtype=U8, device="cuda")
        marks = [both[:, :, i].transpose(0, 1) for i in range(2)]
    else:  # the middle one of three layers
        buf = torch.full((2, n_pages, 3, Hk, page, D), 0x7f, dtype=U8, device="cuda")
        pools = [buf[i, :, 1] for i in range(2)]
        both = torch.full((2, n_pages, 3, Hk, mark), 255, dtype=U8, device="cuda")
        marks = [both[i, :, 1] for i in range(2)]
    return [p.view(FP8) for p in pools] + [m.view(E8M0) for m in marks]


@pytest.mark.parametrize("layout", ["pages", "heads", "layers"])
def test_pools_cut_from_one_buffer(kernels, layout):
    """The same bits as from pools of their own."""
    Hq, Hk, D, page, lens, new = 8, 2, 64, 32, [70, 33, 5], [40, 33, 1]
    g = torch.Generator().manual_seed(3)
    T, n_pages = sum(new), 9
    qkv = torch.randn(T, (Hq + 2 * Hk) * D, generator=g).to(BF16).cuda()
    inv = (1.0 / 1e6 ** (torch.arange(0, D, 2).float() / D)).cuda()
    table = torch.randperm(n_pages, generator=g).view(3, 3).to(torch.int32).cuda()
    dev = torch.tensor(lens, dtype=torch.int32, device="cuda")
    start = torch.tensor([0] + new).cumsum(0).to(torch.int32).cuda()
    old = torch.randint(0, 100, (2, n_pages, Hk, page, D), generator=g).to(U8).cuda()
    results = []
    for cache in (_layers(layout, n_pages, Hk, page, D),
                  [torch.zeros(n_pages, Hk, page, D, dtype=U8, device="cuda").view(FP8) for _ in range(2)] +
                  [torch.zeros(n_pages, Hk, page // 16, dtype=U8, device="cuda").view(E8M0) for _ in range(2)]):
        for i in range(2):
            cache[i].view(U8).copy_(old[i])
            cache[2 + i].view(U8).fill_(120)
        q = kernels.paged_append_fp8(qkv, None, inv, table, dev, *cache, Hq, q_start=start)
        out = kernels.paged_attention_fp8(q, *cache, table, dev, Hq, q_start=start)
        torch.cuda.synchronize()
        results.append([q.view(torch.int16), out.view(torch.int16)] + [t.view(U8).clone() for t in cache])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("Hq,Hk,D,shared,window,sinks", [(28, 4, 128, 0, 0, 0), (14, 2, 64, 0, 50, 3), (28, 4, 128, 64, 0, 0),
                                                         (14, 2, 64, 64, 40, 2)])
@pytest.mark.parametrize("ragged", [True, False])
def test_a_captured_step_of_any_batch(kernels, Hq, Hk, D, shared, window, sinks, ragged):
    """One captured step of append and attention, replayed for other lengths (and numbers of tokens), sequences without
    any and padded rows; eager work between the replays, each of which has to give the eager step's bits."""
    page, B, width = 16, 4, 30
    T = 64 if ragged else B
    g = torch.Generator().manual_seed(D + shared)
    n_pages = B * width
    order = torch.randperm(n_pages, generator=g).view(B, width).to(torch.int32)
    order[:, :shared // page] = order[0, :shared // page]
    table = order.cuda()
    cache = [torch.randint(0, 120, (n_pages, Hk, page, D), generator=g).to(U8).cuda().view(FP8) for _ in range(2)]
    cache += [torch.randint(118, 124, (n_pages, Hk, 1), generator=g).to(U8).cuda().view(E8M0) for _ in range(2)]
    qkv = torch.zeros(T, (Hq + 2 * Hk) * D, dtype=BF16, device="cuda")
    inv = (1.0 / 1e6 ** (torch.arange(0, D, 2).float() / D)).cuda()
    lens = torch.full((B,), shared + 1, dtype=torch.int32, device="cuda")
    start = torch.arange(B + 1, dtype=torch.int32, device="cuda") if ragged else None
    q, out = (torch.zeros(T, Hq * D, dtype=BF16, device="cuda") for _ in range(2))
    work = kernels.paged_attention_fp8_workspace(T, B, Hq, Hk, D, width * page, ragged=ragged, shared=shared)

    def step(q, out, work):
        kernels.paged_append_fp8(qkv, None, inv, table, lens, *cache, Hq, q_start=start, out=q)
        kernels.paged_attention_fp8(q, *cache, table, lens, Hq, q_start=start, shared=shared, window=window, sinks=sinks,
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
        if not ragged:
            new, total = [1] * B, [max(n, shared + 1) for n in total]
        qkv.copy_(torch.randn(qkv.shape, generator=g).to(BF16))
        lens.copy_(torch.tensor(total, dtype=torch.int32))
        if ragged:
            start.copy_(torch.tensor([0] + new).cumsum(0).to(torch.int32))
        q.fill_(7.0)
        out.fill_(7.0)
        before = [t.view(U8).clone() for t in cache]
        graph.replay()
        torch.cuda.synchronize()
        after = [t.view(U8).clone() for t in cache]
        for t, b in zip(cache, before):
            t.view(U8).copy_(b)
        again, mine = torch.full_like(out, 7.0), torch.full_like(q, 7.0)
        step(mine, again, None)
        torch.cuda.synchronize()
        assert torch.equal(again.view(torch.int16), out.view(torch.int16)) and torch.equal(mine, q)
        assert all(torch.equal(t.view(U8), a) for t, a in zip(cache, after))
        assert bool((out[sum(new):] == 7).all())


def test_two_streams(kernels):
    """Two batches at once, each with a workspace of its own."""
    Hq, Hk, D = 28, 4, 128
    batches = [F.Fp8Batch([3000, 700, 5], None, Hk, D, 16, seed=1), F.Fp8Batch([900, 64], [200, 3], Hk, D, 16, seed=2)]
    qs = [_queries(b.T, Hq, D, i) for i, b in enumerate(batches)]
    alone = [_attend(kernels, b, q, Hq) for b, q in zip(batches, qs)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                b = batches[i]
                outs[i].append(kernels.paged_attention_fp8(qs[i], *b.cache(), b.table, b.lens, Hq, q_start=b.q_start))
    torch.cuda.synchronize()
    for got, want in zip(outs, alone):
        assert all(torch.equal(x, want) for x in got)
