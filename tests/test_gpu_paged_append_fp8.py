"""Append to a paged cache in 8 bits: queries, scales, codes, the rows of a block from before, and all the rest as it
was."""
import pytest
import torch

import paged_fp8_ref as F
from paged_fp8_ref import E8M0, FP8

BF16, U8 = torch.bfloat16, torch.uint8
pytestmark = pytest.mark.gpu


class Append:
    """A batch's new tokens over pages of random codes and scales, and what they have to look like afterwards."""

    def __init__(self, Hq, Hk, D, page, lens, new, seed=0, scale=1.0, bias=True, pad=0, first=None):
        g = torch.Generator().manual_seed(seed)
        self.Hq, self.Hk, self.D, self.page, self.lens = Hq, Hk, D, page, lens
        self.new = [1] * len(lens) if new is None else new
        B, H, T = len(lens), Hq + 2 * Hk, sum(self.new)
        width = max(-(-max(n, 1) // page) for n in lens) + 1
        # pages of the new tokens only; the others are not in the pool
        self.table, self.n_pages = torch.full((B, width), -1, dtype=torch.int32), 2
        self.table[::2] = 1 << 30
        order = torch.randperm(sum(self.new) // page + 3 * B + 2, generator=g).tolist()
        for b in range(B):
            for j in range(max(lens[b] - self.new[b], 0) // page, -(-max(lens[b], 0) // page)):
                self.table[b, j] = order[self.n_pages - 2]
                self.n_pages += 1
        self.n_pages = len(order)
        x = torch.randn(T + pad, H * D + 8, generator=g) * scale
        if first is not None:
            x = first(x)
        self.qkv = x.to(BF16).cuda()[:, :H * D]
        self.bias = torch.randn(H * D, generator=g).to(BF16).cuda() if bias else None
        self.inv = (1.0 / 1e6 ** (torch.arange(0, D, 2).float() / D)).cuda()
        codes = torch.randint(0, 256, (2, self.n_pages, Hk, page, D), generator=g).to(U8)
        codes[codes & 127 == 127] = 1
        scales = torch.randint(117, 129, (2, self.n_pages, Hk, page // 16), generator=g).to(U8)
        self.codes, self.scales = codes, scales
        self.pools = [F.strided_codes(c.view(FP8), "cuda") for c in codes]
        self.marks = [F.strided_scales(s.view(E8M0), "cuda") for s in scales]
        self.start = None
        if new is not None:
            self.start = torch.tensor([0] + self.new).cumsum(0).to(torch.int32).cuda()
        self.dev_table, self.dev_lens = self.table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()

    def call(self, kernels, **kw):
        return kernels.paged_append_fp8(self.qkv, self.bias, self.inv, self.dev_table, self.dev_lens, *self.pools,
                                        *self.marks, self.Hq, q_start=self.start, **kw)

    def values(self):
        """Rotated values of all tokens [T, H, D] in float64, and a bound on their error in fp32."""
        T = sum(self.new)
        pos = torch.tensor([self.lens[b] - n + i for b, n in enumerate(self.new) for i in range(n)])
        x = self.qkv[:T].cpu().double() + (self.bias.cpu().double() if self.bias is not None else 0)
        x = x.view(T, self.Hq + 2 * self.Hk, self.D)
        ang = (pos.double()[:, None] * self.inv.cpu().double())[:, None]
        lo, hi = x[:, :self.Hq + self.Hk].chunk(2, -1)
        y = torch.cat([torch.cat([lo * ang.cos() - hi * ang.sin(), hi * ang.cos() + lo * ang.sin()], -1),
                       x[:, self.Hq + self.Hk:]], 1)
        # of the pair's magnitude a few fp32 steps (angle, sine, two products); a value head is the sum alone
        off = x.abs().view(T, -1, 2, self.D // 2).amax(2).repeat(1, 1, 2) * 2.0 ** -19
        off[:, self.Hq + self.Hk:] = x[:, self.Hq + self.Hk:].abs() * 2.0 ** -23
        return y, off

    def check(self, q=None):
        """Of the pools: untouched bytes, scales, codes."""
        y, off = self.values()
        if q is not None:
            err = (q[:y.shape[0]].cpu().double().view(-1, self.Hq, self.D) - y[:, :self.Hq]).abs()
            assert bool((err <= y[:, :self.Hq].abs() * 2.0 ** -8 + off[:, :self.Hq]).all())
        blocks = {}  # (sequence, block) -> its token rows
        t = 0
        for b, n in enumerate(self.new):
            for i in range(n):
                p = self.lens[b] - n + i
                if p >= 0:
                    blocks.setdefault((b, p // 16), []).append((t, p))
                t += 1
        for i in range(2):
            got = self.pools[i].contiguous().view(U8).cpu()
            marks = self.marks[i].contiguous().view(U8).cpu()
            codes, scales = self.codes[i].clone(), self.scales[i].clone()
            for (b, j), rows in blocks.items():
                pg = int(self.table[b, 16 * j // self.page])
                if not 0 <= pg < self.n_pages:
                    continue
                k, held = j % (self.page // 16), rows[0][1] % 16
                z = y[[t for t, _ in rows]][:, self.Hq + i * self.Hk:self.Hq + (i + 1) * self.Hk].transpose(0, 1)
                o = off[[t for t, _ in rows]][:, self.Hq + i * self.Hk:self.Hq + (i + 1) * self.Hk].transpose(0, 1)
                fin = z.abs() <= torch.finfo(torch.float32).max  # (what passes fp32 is infinite there)
                top = torch.where(fin, z.abs(), 0.0).amax((1, 2))
                slack = torch.where(fin, o, 0.0).amax((1, 2))
                old = scales[pg, :, k].int() - 127
                low, high = F.exponent((top - slack).clamp(min=0)), F.exponent(top + slack)
                if held:
                    low, high = torch.maximum(low, old), torch.maximum(high, old)
                e = marks[pg, :, k].int() - 127
                assert bool(((e >= low) & (e <= high)).all()), (e, low, high)
                scales[pg, :, k] = marks[pg, :, k]
                unit = torch.exp2(e.double())[:, None, None]
                at = slice(16 * k, 16 * k + held)
                before = codes[pg, :, at].contiguous().view(FP8).float() * torch.exp2((old - e).float())[:, None, None]
                codes[pg, :, at] = before.to(FP8).view(U8)
                at = slice(16 * k + held, 16 * k + held + len(rows))
                new = got[pg, :, at].contiguous()
                value = new.view(FP8).double() * unit
                assert bool((torch.isnan(value) == ~fin).all())
                want = torch.where(fin, z, 0.0)
                # half a step of e4m3: 2^-4 of the value, 2^-10 of the scale where its range ends; past the range 448
                # of the largest scale
                bound = torch.maximum(want.abs() * 2.0 ** -4, 2.0 ** -10 * unit.expand_as(want)) + o
                want = want.clamp(-448 * 2.0 ** 119, 448 * 2.0 ** 119)
                assert bool(((torch.where(fin, value, 0.0) - want).abs() <= torch.where(fin, bound, 0.0)).all())
                codes[pg, :, at] = new
            assert torch.equal(got, codes) and torch.equal(marks, scales)


@pytest.mark.parametrize("Hq,Hk,D,page,bias", [(28, 4, 128, 16, True), (3, 3, 64, 48, False), (16, 1, 128, 32, True),
                                               (14, 2, 64, 64, True), (16, 16, 128, 16, True)])
@pytest.mark.parametrize("lens,new", [([1, 50, 0, 33], None), ([40, 300000, 2, 16], [40, 7, 5, 0]), ([17], [1]),
                                      ([5 + i for i in range(70)], [i % 4 for i in range(70)]),
                                      ([1500, 33, 700], [1400, 2, 333])])
def test_append(kernels, Hq, Hk, D, page, bias, lens, new):
    a = Append(Hq, Hk, D, page, lens, new, seed=D + len(lens), bias=bias, pad=0 if new is None else 4)
    out = torch.full((a.qkv.shape[0], Hq * D), 7.0, dtype=BF16, device="cuda")
    assert a.call(kernels, out=out) is out
    torch.cuda.synchronize()
    T = sum(a.new)
    assert bool((out[T:] == 7).all())
    a.check(out)


@pytest.mark.parametrize("scale", [2.0 ** -126, 2.0 ** -60, 1e-3, 300.0, 2.0 ** 100, 2.0 ** 126])
@pytest.mark.parametrize("D", [64, 128])
def test_magnitudes(kernels, scale, D):
    """Scales at both ends of their range, and rows from before that grow or shrink beside them."""
    a = Append(4, 2, D, 16, [30, 5, 90, 17], [3, 1, 20, 1], seed=1, scale=scale, bias=False)
    a.call(kernels)
    torch.cuda.synchronize()
    a.check()


def test_zeros_nan_and_infinities(kernels):
    """Zeros alone; NaN and infinities, which neither count for the scale nor touch other values."""
    def first(x):
        x[0] = 0.0
        x[1, 5 * 128 + 3] = float("nan")
        x[2, 4 * 128:4 * 128 + 20] = float("inf")
        x[2, 7 * 128 + 70] = float("-inf")
        x[3] = float("nan")
        return x
    a = Append(4, 2, 128, 16, [1, 50, 20, 33], [1, 1, 1, 1], seed=2, bias=False, first=first)
    a.call(kernels)
    torch.cuda.synchronize()
    y, _ = a.values()
    assert not bool(torch.isfinite(y[2, 4, :20]).any())
    # (a pair with an infinity turns into infinities and NaN, neither of which is finite)
    a.check()


@pytest.mark.parametrize("D", [64, 128])
def test_token_by_token_and_at_once(kernels, D):
    """A sequence appended in one call, in odd chunks and token by token: the same scales, and codes that differ where
    an early one was rounded to a smaller scale first, by a second rounding at most."""
    Hq, Hk, page, n = 4, 2, 32, 77
    g = torch.Generator().manual_seed(D)
    qkv = (torch.randn(n, (Hq + 2 * Hk) * D, generator=g) * torch.exp2(torch.randint(-3, 4, (n, 1), generator=g).float())
           ).to(BF16).cuda()
    inv = (1.0 / 1e6 ** (torch.arange(0, D, 2).float() / D)).cuda()
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    got = []
    for chunks in ([n], [1] * n, [5, 20, 1, 1, 3, 40, 7]):
        k, v = (torch.full((3, Hk, page, D), 0x7f, dtype=U8, device="cuda").view(FP8) for _ in range(2))
        ks, vs = (torch.full((3, Hk, page // 16), 255, dtype=U8, device="cuda").view(E8M0) for _ in range(2))
        at = 0
        for c in chunks:
            start = torch.tensor([0, c], dtype=torch.int32, device="cuda")
            kernels.paged_append_fp8(qkv[at:at + c], None, inv, table,
                                     torch.tensor([at + c], dtype=torch.int32, device="cuda"), k, v, ks, vs, Hq,
                                     q_start=start if c > 1 else None)
            at += c
        torch.cuda.synchronize()
        got.append((k, v, ks, vs))
    for other in got[1:]:
        for x, y in zip(got[0][2:], other[2:]):
            assert torch.equal(x.view(U8), y.view(U8))
        for pool, scales, mine in zip(got[0][:2], got[0][2:], other[:2]):
            x, y = (p[table[0].long()].transpose(0, 1).reshape(Hk, -1, D)[:, :n].view(U8).view(FP8).double()
                    for p in (pool, mine))
            # half a step each, and the second one's of the first's result: in codes, with a step of 2^-9 at least
            step = torch.maximum(torch.maximum(x.abs(), y.abs()) * 2.0 ** -3, torch.full_like(x, 2.0 ** -9))
            assert bool(((x - y).abs() <= step).all())


def test_entries_outside_the_pool_and_rows_of_no_sequence(kernels):
    """Sequences without a page for some of their tokens, rows before and behind the batch's."""
    a = Append(4, 2, 64, 16, [40, 20, 70], [30, 4, 50], seed=6)
    a.table[0, 1] = -5
    a.table[2, 3] = a.n_pages
    a.dev_table.copy_(a.table)
    a.call(kernels)
    torch.cuda.synchronize()
    a.check()
