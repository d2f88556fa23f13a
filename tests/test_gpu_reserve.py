"""Kernels.paged_reserve against a list per sequence and a Python stack."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


class Model:
    """The stack and every sequence's pages as lists; ``change`` as paged_reserve documents it."""

    def __init__(self, B, width, page, n_pages, capacity, seed, strided=True):
        self.rng = random.Random(seed)
        self.B, self.width, self.page, self.capacity = B, width, page, capacity
        order = list(range(n_pages))
        self.rng.shuffle(order)
        self.free = order + [-7] * (capacity - n_pages)
        self.n_free = n_pages
        self.table = [[-1] * width for _ in range(B)]
        self.lens = [0] * B
        self.dev = {"lens": torch.zeros(B, dtype=torch.int32, device="cuda"),
                    "free": torch.tensor(self.free, dtype=torch.int32, device="cuda"),
                    "n_free": torch.tensor([n_pages], dtype=torch.int32, device="cuda")}
        buf = torch.full((B, width + (3 if strided else 0)), -1, dtype=torch.int32, device="cuda")
        self.dev["pages"] = buf[:, :width]
        self.buf = buf

    def change(self, new, rows):
        """(q_start, slots, short), and the state after it."""
        ps = self.page
        total = [min(max(n, 0), self.width * ps) + d for n, d in zip(self.lens, new)]
        total = [max(n, 0) for n in total]
        had, has = ([-(-n // ps) for n in ns] for ns in (self.lens, total))
        held = [min(h, self.width) for h in has]
        taken = sum(max(h - o, 0) for h, o in zip(held, had))
        given = sum(max(o - h, 0) for h, o in zip(held, had))
        short = max(taken - self.n_free - given, 0)
        tokens = sum(max(n, 0) for n in new)
        bad = short > 0 or any(n > self.width * ps for n in total) or self.n_free + given > self.capacity
        bad |= rows is not None and tokens > rows
        if bad:
            return [0] * (self.B + 1), None if rows is None else [-1] * rows, short if short else -1
        back = [self.table[b][j] for b in range(self.B) for j in range(has[b], had[b])]
        for p in reversed(back):
            self.free[self.n_free] = p
            self.n_free += 1
        for b in range(self.B):
            for j in range(had[b], has[b]):
                self.n_free -= 1
                self.table[b][j] = self.free[self.n_free]
        start, slots = [0], []
        for b in range(self.B):
            n = max(new[b], 0)
            start.append(start[-1] + n)
            slots += [self.table[b][p // ps] * ps + p % ps for p in range(total[b] - n, total[b])]
        self.lens = total
        return start, None if rows is None else slots + [-1] * (rows - len(slots)), 0

    def check(self, got, want):
        torch.cuda.synchronize()
        q_start, slots, short = got
        assert q_start.tolist() == want[0] and short.tolist() == [want[2]]
        assert (slots is None) == (want[1] is None)
        if slots is not None:
            assert slots.dtype == torch.int64 and slots.tolist() == want[1]
        assert self.dev["lens"].tolist() == self.lens and self.dev["n_free"].tolist() == [self.n_free]
        assert self.dev["free"].tolist() == self.free and self.dev["pages"].tolist() == self.table
        assert bool((self.buf[:, self.width:] == -1).all())


def _call(kernels, m, new, rows, **kw):
    return kernels.paged_reserve(torch.tensor(new, dtype=torch.int32, device="cuda"), m.dev["lens"], m.dev["pages"],
                                 m.dev["free"], m.dev["n_free"], m.page, rows=rows, **kw)


@pytest.mark.parametrize("B,page,most", [(1, 16, 1), (1, 16, 500), (3, 48, 100), (64, 16, 40), (65, 64, 300), (1000, 16, 20),
                                         (1024, 32, 9), (1025, 16, 33), (2500, 16, 12)])
def test_grow_and_shrink(kernels, B, page, most):
    """Steps of growing and shrinking sequences, empty ones among them; steps that take everything back restore the stack."""
    width = 3 * -(-most // page) + 2
    m = Model(B, width, page, B * width, B * width + 5, seed=B)
    for step in range(6):
        rng = m.rng
        new = [rng.choice([0, 1, rng.randint(0, most), -rng.randint(0, most) if step else 1]) for _ in range(B)]
        if step == 4:
            new = [-n for n in m.lens]
        rows = rng.choice([None, sum(max(n, 0) for n in new), sum(max(n, 0) for n in new) + 70])
        before = (list(m.free[:m.n_free]), m.n_free)
        got = _call(kernels, m, new, rows)
        m.check(got, m.change(new, rows))
        if all(n >= 0 for n in new):
            back = [-n for n in new]
            got = _call(kernels, m, back, None)
            m.check(got, m.change(back, None))
            assert (m.free[:m.n_free], m.n_free) == before
            got = _call(kernels, m, new, rows)
            m.check(got, m.change(new, rows))


@pytest.mark.parametrize("B,tokens", [(1, 4000), (1, 4200), (1, 8192), (1, 8193), (40, 1000), (1100, 30)])
def test_many_rows(kernels, B, tokens):
    """Slot maps on both sides of the launch of their own, and one behind which rows are left."""
    m = Model(B, tokens // 16 + 3, 16, B * (tokens // 16 + 3), B * (tokens // 16 + 3), seed=tokens)
    for new in ([7] * B, [tokens - b % 3 for b in range(B)]):
        rows = sum(new) + 100
        m.check(_call(kernels, m, new, rows), m.change(new, rows))


@pytest.mark.parametrize("B", [5, 1500])
@pytest.mark.parametrize("why", ["pages", "width", "rows", "capacity", "exactly enough"])
def test_as_a_whole_or_not_at_all(kernels, B, why):
    m = Model(B, 4, 16, 3 * B, 3 * B, seed=3)
    new = [20] * B
    m.check(_call(kernels, m, new, None), m.change(new, None))
    assert m.n_free == B
    new, rows = [1] * B, B
    if why == "pages":
        new, rows = [20] * B, 100 * B  # 36 ..  40 positions: a page each, and two of them one more
        new[0] = new[B - 1] = 29
    elif why == "width":
        new[B - 1], rows = 45, 100 * B
    elif why == "rows":
        rows = B - 1
    elif why == "capacity":
        m.capacity -= 1  # (the stack has B, 2 B come back)
        m.dev["free"], m.free = m.dev["free"][:-1], m.free[:-1]
        new, rows = [-20] * B, 4
    else:
        new, rows = [20] * B, 20 * B
    want = m.change(new, rows)
    assert want[2] == {"pages": 2, "exactly enough": 0}.get(why, -1)
    m.check(_call(kernels, m, new, rows), want)
    # and the batch goes on
    new = [0] * (B - 1) + [1]
    m.check(_call(kernels, m, new, 3), m.change(new, 3))


def test_pages_given_back_serve_the_same_call(kernels):
    m = Model(3, 8, 16, 8, 8, seed=9)
    for new in ([100, 20, 0], [-100, 100, 0], [5, -70, 60], [-5, -50, -60]):
        m.check(_call(kernels, m, new, 200), m.change(new, 200))
    assert m.n_free == 8


def test_captured_steps(kernels):
    """One captured call replayed with other counts, between eager work, into buffers that are handed over."""
    B = 9
    m = Model(B, 12, 16, 60, 70, seed=4)
    new = torch.zeros(B, dtype=torch.int32, device="cuda")
    out = (torch.empty(B + 1, dtype=torch.int32, device="cuda"), torch.empty(200, dtype=torch.int64, device="cuda"),
           torch.empty(1, dtype=torch.int32, device="cuda"))

    def call():
        return kernels.paged_reserve(new, m.dev["lens"], m.dev["pages"], m.dev["free"], m.dev["n_free"], 16, rows=200, out=out)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert call() is out  # (counts of zero: nothing changes)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for step in range(7):
        counts = [m.rng.randint(-20, 40) for _ in range(B)] if step != 3 else [190] * B
        new.copy_(torch.tensor(counts, dtype=torch.int32))
        graph.replay()
        m.check(out, m.change(counts, 200))
