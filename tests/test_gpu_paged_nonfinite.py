"""ns_paged_attention with NaN and infinities: in what a token sees they come out as the formula says, whatever
path and split the call takes; in what no token sees they have no effect."""
import math

import pytest
import torch

import paged_ref as R

BF16 = torch.bfloat16
NAN, INF = float("nan"), float("inf")
pytestmark = pytest.mark.gpu

LAYOUTS = [(28, 4, 128), (14, 2, 64), (40, 2, 128)]
# (lens, new, shared): single tokens of one range and of many, prompts of one range and of many, both behind a
# prefix that all share
BATCHES = {
    "one": ([5, 40, 700, 3000, 0, 64], None, 0),
    "one long": ([9000], None, 0),
    "tiles": ([60, 17], [60, 3], 0),
    "tiles split": ([1000, 40], [300, 40], 0),
    "one shared": ([700, 130, 90, 101], None, 100),
    "tiles shared": ([641, 900, 640], [1, 90, 4], 640),
}


def _queries(T, Hq, D, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, Hq * D, generator=g) * 2).to(BF16).cuda()


def formula(batch, q, Hq, window=0, sinks=0, hidden=None):
    """[T, Hq, D] float64: the softmax over the keys that a token sees, taken out of the others, of any values.
    hidden(b, positions): positions left out besides."""
    D, rep = batch.D, Hq // batch.Hk
    q = q.cpu().double().view(-1, Hq, D)
    out = torch.zeros(batch.T, Hq, D, dtype=torch.float64)
    kv = {}
    for t, b, p in batch.rows():
        if b not in kv:
            n = max(batch.host_lens[b], 0)
            kv[b] = batch.gather(batch.k, b, n), batch.gather(batch.v, b, n), torch.arange(n)
        k, v, j = kv[b]
        see = j <= p
        if window:
            see &= (j > p - window) | (j < sinks)
        if hidden is not None:
            see &= ~hidden(b, j)
        if bool(see.any()):
            for g in range(batch.Hk):
                s = q[t, g * rep:(g + 1) * rep] @ k[g][see].t() * D ** -0.5
                out[t, g * rep:(g + 1) * rep] = torch.softmax(s, -1) @ v[g][see]
    return out


def _check(got, want, v_max=8.0):
    """Half a bf16 step of the result (2^-8 of it), and of the largest finite value: 2^-16 for the probabilities'
    two terms and 2^-14 for fp32 scores up to a few hundred in the exponent. NaN where the formula has it."""
    got = got.cpu().double().view_as(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    err = (got - want).abs().nan_to_num(0.0)
    bound = want.abs().nan_to_num(0.0) * 2.0 ** -8 + 2.0 ** -13 * v_max
    assert bool((err <= bound).all()), float((err - bound).max())


def _batch(name, Hk, D):
    lens, new, shared = BATCHES[name]
    return R.PagedBatch(lens, new, Hk, D, 16, shared=shared, seed=7), shared


def _set(batch, pool, b, j, value, dim=slice(None)):
    pool[int(batch.cpu_table[b, j // batch.page]), :, j % batch.page, dim] = value


def _attend(kernels, batch, q, Hq, shared, **kw):
    got = kernels.paged_attention(q, batch.k, batch.v, batch.table, batch.lens, Hq, q_start=batch.q_start,
                                  shared=shared, **kw)
    torch.cuda.synchronize()
    return got


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("name", BATCHES)
def test_nan_query(kernels, name, Hq, Hk, D):
    """A NaN in a query head makes that token's head NaN, and nothing else."""
    batch, shared = _batch(name, Hk, D)
    q = _queries(batch.T, Hq, D, 1)
    for t in range(0, batch.T, max(batch.T // 3, 1)):
        q[t, (t * 5 % Hq) * D + t % D] = NAN
    want = formula(batch, q, Hq)
    assert bool(torch.isnan(want).any())
    _check(_attend(kernels, batch, q, Hq, shared), want)


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("where", ["one", "first half", "all but the last"])
def test_nan_keys(kernels, name, where, Hq, Hk, D):
    """NaN keys, one or as many as fill whole ranges of the work, reach every token that sees one of them."""
    batch, shared = _batch(name, Hk, D)
    n = batch.host_lens[0]
    lo, hi = {"one": (n // 2, n // 2 + 1), "first half": (0, n // 2), "all but the last": (0, n - 1)}[where]
    for j in range(lo, hi):
        _set(batch, batch.k, 0, j, NAN)
    q = _queries(batch.T, Hq, D, 2)
    want = formula(batch, q, Hq)
    assert bool(torch.isnan(want).any())
    _check(_attend(kernels, batch, q, Hq, shared), want)


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("name", BATCHES)
@pytest.mark.parametrize("where", ["one", "first half", "last half", "all"])
def test_infinite_scores(kernels, name, where, Hq, Hk, D):
    """Scores of -inf weigh nothing beside finite ones, and are NaN where a token sees no other; +inf is NaN."""
    batch, shared = _batch(name, Hk, D)
    q = _queries(batch.T, Hq, D, 3)
    q[:, ::D] = 1.0
    n = batch.host_lens[0]
    lo, hi = {"one": (n // 2, n // 2 + 1), "first half": (0, n // 2), "last half": (n // 2, n), "all": (0, n)}[where]
    for j in range(lo, hi):
        _set(batch, batch.k, 0, j, -INF, 0)
    want = formula(batch, q, Hq)
    assert where != "all" or bool(torch.isnan(want).any())
    _check(_attend(kernels, batch, q, Hq, shared), want)
    for j in range(lo, hi):
        _set(batch, batch.k, 0, j, INF, 0)
    want = formula(batch, q, Hq)
    assert bool(torch.isnan(want).any())
    _check(_attend(kernels, batch, q, Hq, shared), want)


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("name", BATCHES)
def test_nan_and_infinite_values(kernels, name, Hq, Hk, D):
    """A NaN or infinite value that a token sees never leaves that dimension of its output finite; the other
    dimensions keep theirs."""
    for value in (NAN, INF, -INF):
        batch, shared = _batch(name, Hk, D)
        q = _queries(batch.T, Hq, D, 4)
        want = formula(batch, q, Hq)
        at = batch.host_lens[0] // 2
        _set(batch, batch.v, 0, at, value, 3)
        got = _attend(kernels, batch, q, Hq, shared).cpu().double().view_as(want)
        sees = [(b == 0 or at < shared) and p >= at for _, b, p in batch.rows()]
        assert any(sees)
        assert not bool(torch.isfinite(got[sees][..., 3]).any())
        rest = [d for d in range(D) if d != 3]
        _check(got[..., rest], want[..., rest])


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
def test_nothing_seen_beside_nan(kernels, Hq, Hk, D):
    """Tokens that see nothing get zeros beside NaN queries and keys: no positions, more new tokens than
    positions, all of a sequence's pages outside the pool."""
    q = _queries(40, Hq, D, 5)
    q[::2] = NAN
    batch = R.PagedBatch([0, 50, 16, 0], None, Hk, D, 16, seed=2)
    batch.table[2] = -1
    got = _attend(kernels, batch, q[:4], Hq, 0).view(4, Hq, D)
    assert bool((got[[0, 2, 3]] == 0).all()) and bool(torch.isfinite(got[1]).all())
    for shared in (0, 2):
        batch = R.PagedBatch([2, 20, 2], [6, 20, 2], Hk, D, 16, shared=shared, seed=3)
        got = _attend(kernels, batch, q[:28], Hq, shared).view(28, Hq, D)
        assert bool((got[:4] == 0).all())
        assert bool(torch.isnan(got[4:28:2]).all()) and bool(torch.isfinite(got[5:28:2]).all())


# ------------------------------------------------------------------ a shared prefix seen through windows
# Sequences whose windows end inside the prefix, or begin past it: the positions between them are seen by none.
@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("sinks", [0, 3, 70])
@pytest.mark.parametrize("lens,new,shared", [
    ([300, 1000], None, 900), ([300, 1000, 650], None, 1000), ([64, 2000, 130, 64], None, 1500),
    ([300, 1000, 420], [3, 1, 40], 900), ([1300, 200, 700], [1, 4, 30], 1200), ([1000, 990, 1100], None, 900)])
def test_shared_window_gaps(kernels, lens, new, shared, sinks, Hq, Hk, D):
    window = 60
    batch = R.PagedBatch(lens, new, Hk, D, 16, shared=shared, seed=sinks)
    seen = torch.zeros(max(lens), dtype=torch.bool)
    for _, b, p in batch.rows():
        j = torch.arange(max(lens))
        seen |= (j <= p) & ((j > p - window) | (j < sinks))
    at = lens.index(max(lens))
    gone = [j for j in range(min(shared, max(lens))) if not seen[j]]
    assert gone
    q = _queries(batch.T, Hq, D, 6)
    want = formula(batch, q, Hq, window, sinks)
    for value in (NAN, INF):
        for j in gone:
            for pool in (batch.k, batch.v):
                _set(batch, pool, at, j, value)
        _check(_attend(kernels, batch, q, Hq, shared, window=window, sinks=sinks), want)


# ------------------------------------------------------------------ padding and bad tables behind a shared prefix
@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 2)])
@pytest.mark.parametrize("lens,new,shared", [([150, 140, 103], [10, 40, 3], 100), ([700, 650, 640], [2, 1, 0], 640),
                                             ([3, 90, 2], [8, 20, 5], 64)])
def test_shared_prefix_with_rows_of_no_sequence(kernels, lens, new, shared, window, sinks, Hq, Hk, D):
    """Rows behind the last sequence keep what they hold and do not reach the others, also where they are NaN;
    more new tokens than positions see nothing."""
    batch = R.PagedBatch(lens, new, Hk, D, 16, shared=shared, seed=1)
    T = batch.T + 60
    q = _queries(T, Hq, D, 3)
    q[batch.T:] = NAN
    out = torch.full((T, Hq * D), 7.0, dtype=BF16, device="cuda")
    kernels.paged_attention(q, batch.k, batch.v, batch.table, batch.lens, Hq, q_start=batch.q_start, out=out,
                            shared=shared, window=window, sinks=sinks)
    assert bool((out[batch.T:] == 7).all())
    _check(out[:batch.T], formula(batch, q[:batch.T], Hq, window, sinks))


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("new", [None, [3, 40, 1]])
def test_entries_outside_the_pool_in_a_shared_prefix(kernels, new, Hq, Hk, D):
    """Their positions are left out for every sequence."""
    batch = R.PagedBatch([300, 350, 290], new, Hk, D, 16, shared=256, seed=5)
    q = _queries(batch.T, Hq, D, 7)
    for entry in (-1, batch.k.shape[0], (1 << 31) - 1):
        for pages in ([0], [3, 4], list(range(16))):
            table = batch.table.clone()
            table[:, pages] = entry
            want = formula(batch, q, Hq, hidden=lambda b, j: torch.isin(j // 16, torch.tensor(pages)))
            got = kernels.paged_attention(q, batch.k, batch.v, table, batch.lens, Hq, q_start=batch.q_start, shared=256)
            _check(got, want)


@pytest.mark.parametrize("Hq,Hk,D", LAYOUTS)
@pytest.mark.parametrize("lens,new,shared", [([300, 700], None, 0), ([300, 700], [40, 300], 0), ([300, 350], [3, 40], 256),
                                             ([300, 350], None, 256)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (50, 20)])
def test_scores_that_are_all_minus_infinity_beside_entries_outside_the_pool(kernels, lens, new, shared, window, sinks,
                                                                            Hq, Hk, D):
    """NaN where a page is there, 0 where all that a token would see is outside the pool."""
    batch = R.PagedBatch(lens, new, Hk, D, 16, shared=shared, seed=5)
    q = _queries(batch.T, Hq, D, 7)
    q[:, ::D] = 1.0
    batch.k[..., 0] = -INF
    width = batch.table.shape[1]
    for pages in ([0], [0, 1, 2, 3, 4, 5, 6, 7], list(range(8, 16)), list(range(18)), list(range(width))):
        table = batch.table.clone()
        table[:, [p for p in pages if p < width]] = -1
        want = formula(batch, q, Hq, window, sinks, hidden=lambda b, j: torch.isin(j // 16, torch.tensor(pages)))
        got = kernels.paged_attention(q, batch.k, batch.v, table, batch.lens, Hq, q_start=batch.q_start, shared=shared,
                                      window=window, sinks=sinks)
        _check(got, want)
