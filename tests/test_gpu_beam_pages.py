"""Pages that beam search leaves, back on the stack of free pages: Kernels.paged_reorder with the stack against lists, and loops
of reorderings and reservations after which every page is in a row or on the stack, and at the end on the stack."""
import pytest
import torch

from beam_pages_ref import dropped
from nanoserve_amd.qwen import Qwen2Runner, Qwen2Shape
from test_gpu_beam_decode import Server

BF16, I32 = torch.bfloat16, torch.int32
pytestmark = pytest.mark.gpu


def _ints(values):
    return torch.tensor(values, dtype=I32, device="cuda")


def _tree(R, beams, lens, page, groups, seed):
    """Rows [R * beams][width] whose columns a request's beams share in up to `groups` groups, a page of its own for each beam
    behind them; and the number of pages."""
    g = torch.Generator().manual_seed(seed)
    width = max(lens) // page + 2
    kind = torch.randint(0, groups, (R, width, beams), generator=g)
    kind[:, ::3] = 0  # (columns that all share among them)
    ids, table = {}, []
    for r in range(R):
        for i in range(beams):
            row = []
            for j in range(width):
                key = (r, j, int(kind[r, j, i])) if j < lens[r] // page else (r, j, "own", i)
                row.append(ids.setdefault(key, len(ids)))
            table.append(row)
    order = torch.randperm(len(ids), generator=g).tolist()
    return [[order[x] for x in row] for row in table], len(ids)


def _pool(n_pages, page, layers=1, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(-30000, 30000, (layers, n_pages, 2, page, 64), generator=g, dtype=torch.int16).cuda().view(BF16)
            for _ in range(2)]


@pytest.mark.parametrize("R,beams,page,lens,groups", [
    (1, 1, 16, [40], 1), (1, 2, 16, [33], 2), (3, 4, 16, [70, 64, 5], 3), (2, 8, 32, [4000, 100], 8), (1, 64, 16, [1100], 40),
    (40, 5, 16, [16 * (i % 7) + i for i in range(40)], 3), (1, 4, 16, [64 * 64 + 9], 4), (17, 3, 48, [500] * 17, 2)])
def test_dropped_pages(kernels, R, beams, page, lens, groups):
    table, n_pages = _tree(R, beams, lens, page, groups, seed=beams)
    rows = [n for n in lens for _ in range(beams)]
    wide = torch.full((R * beams, len(table[0]) + 3), -7, dtype=I32)
    wide[:, :-3] = torch.tensor(table)
    pages, dev_lens = wide.cuda()[:, :-3], _ints(rows)
    pools = _pool(n_pages, page)
    capacity = n_pages + 9
    g = torch.Generator().manual_seed(R)
    for k in range(6):
        cand = torch.randint(0, beams, (R, beams + 2), generator=g)
        if k == 1:
            cand[:] = beams - 1
        elif k == 2:
            cand[:, :beams] = torch.arange(beams)
        elif k == 3:
            cand[:, :beams] = beams // 2
            cand[:, 0] = -1
        cand = cand.to(I32).cuda()
        parents = cand[:, :beams]
        want = dropped(table, parents.tolist(), rows, page, n_pages)
        height = [0, 9, -3, 4, capacity - len(want), 5][k]
        free = torch.arange(capacity, dtype=I32, device="cuda") + (1 << 20)
        was, n_free = free.clone(), _ints([height])
        other = [p.clone() for p in pools]
        got = kernels.paged_reorder(parents, pages, dev_lens, *pools, free=free, n_free=n_free)
        plain = kernels.paged_reorder(parents, pages, dev_lens, *other)
        torch.cuda.synchronize()
        height = max(height, 0)
        assert int(n_free) == height + len(want)
        was[height:height + len(want)] = _ints(want)
        assert torch.equal(free, was)
        assert torch.equal(got, plain) and all(torch.equal(a.view(torch.int16), b.view(torch.int16)) for a, b in zip(pools, other))
        # what was in a row is in one of the new ones or pushed
        def whole(t):
            return {t[i][j] for i in range(R * beams) for j in range(rows[i] // page)}
        assert whole(table) == whole(got.tolist()) | set(want) and not whole(got.tolist()) & set(want)


def test_stacks_without_room(kernels):
    """A height past the capacity, room for some, and entries that are no pages."""
    table, n_pages = _tree(2, 6, [200, 170], 16, 5, seed=3)
    table[1][2], table[7][3], table[3][0] = -1, n_pages, 1 << 30
    rows = [200] * 6 + [170] * 6
    parents = [[0, 0, 0, 2, 2, 2], [5, 5, 5, 5, 5, 5]]
    want = dropped(table, parents, rows, 16, n_pages)
    assert len(want) > 8
    pools = _pool(n_pages, 16)
    for capacity, height, pushed in ((20, 21, 0), (20, 20, 0), (20, 17, 3), (0, 0, 0), (400, 0, len(want))):
        free = torch.full((capacity + 5,), -9, dtype=I32, device="cuda")
        was, n_free = free.clone(), _ints([height])
        kernels.paged_reorder(_ints(parents), _ints(table), _ints(rows), *pools, free=free[:capacity], n_free=n_free)
        torch.cuda.synchronize()
        assert int(n_free) == height + pushed
        was[height:height + pushed] = _ints(want[:pushed])
        assert torch.equal(free, was)


def _accounted(pages, lens, page, free, n_free, n_pages):
    """Every page is on the stack once or in a row; returns how many are on the stack."""
    rows = pages.tolist()
    used = {rows[i][j] for i, n in enumerate(lens.tolist()) for j in range(-(-n // page))}
    stack = free[:int(n_free)].tolist()
    assert len(set(stack)) == len(stack) and not used & set(stack)
    assert used | set(stack) == set(range(n_pages))
    return len(stack)


def _end(kernels, pages, lens, pools, free, n_free, page, R, beams):
    """Requests end: all beams go on from the first, which drops all other whole pages; then the first gives back everything
    and the others their last pages."""
    pages = kernels.paged_reorder(torch.zeros(R, beams, dtype=I32, device="cuda"), pages, lens, *pools, free=free, n_free=n_free)
    new = -(lens % page)
    new[::beams] = -lens[::beams]
    _, _, short = kernels.paged_reserve(new, lens, pages, free, n_free, page)
    lens.zero_()
    assert int(short) == 0
    return pages


@pytest.mark.parametrize("R,beams,page,start,steps", [(1, 8, 16, 0, 150), (3, 4, 32, 45, 100), (2, 64, 16, 16, 40)])
def test_no_page_is_lost(kernels, R, beams, page, start, steps):
    """A prompt's pages shared by all beams, then steps of random parents and one token each."""
    rows = R * beams
    width = -(-(start + steps) // page) + 1
    n_pages = rows * width
    g = torch.Generator().manual_seed(beams)
    pages = torch.full((rows, width), -1, dtype=I32, device="cuda")
    lens = torch.zeros(rows, dtype=I32, device="cuda")
    free, n_free = torch.randperm(n_pages, generator=g).to(I32).cuda(), _ints([n_pages])
    pools = _pool(n_pages, page)
    new = torch.zeros(rows, dtype=I32, device="cuda")
    new[::beams] = start
    kernels.paged_reserve(new, lens, pages, free, n_free, page)
    whole = start // page
    kernels.paged_reserve(torch.where(new > 0, 0, start % page).to(I32), lens, pages, free, n_free, page)
    own = pages[:, 0].clone()
    for r in range(R):
        others = slice(r * beams + 1, (r + 1) * beams)
        pages[others, :whole] = pages[r * beams, :whole].clone()
        if start % page:
            pages[others, whole] = own[others]
    lens.fill_(start)
    left = _accounted(pages, lens, page, free, n_free, n_pages)
    for step in range(steps):
        parents = torch.randint(0, beams, (R, beams), generator=g).to(I32).cuda()
        pages = kernels.paged_reorder(parents, pages, lens, *pools, free=free, n_free=n_free)
        _accounted(pages, lens, page, free, n_free, n_pages)
        _, _, short = kernels.paged_reserve(torch.ones_like(lens), lens, pages, free, n_free, page)
        assert int(short) == 0
        now = _accounted(pages, lens, page, free, n_free, n_pages)
    # (random parents: hardly more than a few pages of each beam are its own)
    assert left - now < R * (steps // page + 8 * beams)
    _end(kernels, pages, lens, pools, free, n_free, page, R, beams)
    assert int(n_free) == n_pages and sorted(free.tolist()) == list(range(n_pages))


def test_captured(kernels):
    """A captured step (reorder, reserve) replayed with other parents, against the same calls made one by one."""
    R, beams, page, width = 2, 4, 16, 8
    rows, n_pages = R * beams, 2 * 4 * 8
    pools = _pool(n_pages, page)

    def state():
        pages = torch.full((rows, width), -1, dtype=I32, device="cuda")
        s = dict(pages=pages, lens=torch.zeros(rows, dtype=I32, device="cuda"),
                 free=torch.arange(n_pages, dtype=I32, device="cuda"), n_free=_ints([n_pages]), pools=[p.clone() for p in pools],
                 parents=torch.zeros(R, beams, dtype=I32, device="cuda"), out=torch.empty_like(pages))
        s["kept"] = (torch.zeros(rows + 1, dtype=I32, device="cuda"), None, _ints([0]))
        return s

    one = torch.ones(rows, dtype=I32, device="cuda")

    def step(s):
        kernels.paged_reorder(s["parents"], s["pages"], s["lens"], *s["pools"], out=s["out"], free=s["free"], n_free=s["n_free"])
        s["pages"].copy_(s["out"])
        kernels.paged_reserve(one, s["lens"], s["pages"], s["free"], s["n_free"], page, out=s["kept"])

    a, b, warm = state(), state(), state()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a)
    g = torch.Generator().manual_seed(1)
    for k in range(90):
        parents = torch.randint(0, beams, (R, beams), generator=g).to(I32)
        for s in (a, b):
            s["parents"].copy_(parents)
        graph.replay()
        step(b)
        torch.cuda.synchronize()
        for name in ("pages", "lens", "free", "n_free", "out"):
            assert torch.equal(a[name], b[name]), (k, name)
        assert int(a["kept"][2]) == 0
        _accounted(a["pages"], a["lens"], page, a["free"], a["n_free"], n_pages)


def test_beam_search_gives_back_every_page(kernels):
    """A batch of beams over the 8-bit cache, as the operators are used together: no step loses a page, and when its requests end
    all are on the stack."""
    beams, page, lengths, steps = 4, 16, [5, 33, 48], 40
    shape = Qwen2Shape(layers=2, hidden=512, heads=4, kv_heads=2, intermediate=1024, vocab=2000)
    r = Qwen2Runner.random(shape, seed=4, kernels=kernels)
    g = torch.Generator().manual_seed(3)
    R, rows = len(lengths), len(lengths) * beams
    width = (max(lengths) + steps) // page + 2
    n_pages = rows * width
    server = Server(r, rows, width, page, n_pages, seed=1)
    new = torch.zeros(rows, dtype=I32)
    new[::beams] = torch.tensor(lengths, dtype=I32)
    tokens = torch.randint(0, shape.vocab, (sum(lengths),), generator=g).cuda()
    q_start, _ = server.reserve(new, rows=len(tokens))
    logits = server.forward(tokens, q_start)
    part = torch.tensor([n % page for n in lengths], dtype=I32).repeat_interleave(beams)
    part[::beams] = 0
    server.reserve(part)
    own = server.pages[:, 0].clone()
    for i, n in enumerate(lengths):
        others, w = slice(i * beams + 1, (i + 1) * beams), n // page
        server.pages[others, :w] = server.pages[i * beams, :w].clone()
        if n % page:
            server.pages[others, w] = own[others]
        server.lens[i * beams:(i + 1) * beams] = n
    scores = torch.full((R, beams), float("-inf"), device="cuda")
    scores[:, 0] = 0.0
    last = logits[q_start[1:].long()[::beams] - 1].repeat_interleave(beams, 0)
    pools = (server.k, server.v, server.ks, server.vs)
    for _ in range(steps):
        picked, chosen, parents = kernels.beam_select(last, scores, 2 * beams)
        scores = picked[:, :beams].contiguous()
        server.pages = kernels.paged_reorder(parents[:, :beams], server.pages, server.lens, *pools, free=server.free,
                                             n_free=server.n_free)
        server.reserve([1] * rows)
        _accounted(server.pages, server.lens, page, server.free, server.n_free, n_pages)
        last = server.forward(chosen[:, :beams].reshape(-1).long())
    _end(kernels, server.pages, server.lens, pools, server.free, server.n_free, page, R, beams)
    assert int(server.n_free) == n_pages and sorted(server.free.tolist()) == list(range(n_pages))
