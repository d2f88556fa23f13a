"""A batch over a paged cache in plain float64, for the tests of the paged operators."""
import math

import torch

BF16 = torch.bfloat16
NAN = float("nan")


class PagedBatch:
    """Random pools and tables of sequences with ``lens`` positions, ``new`` of them new tokens (None:
    one each). Every pool row that is no position of a sequence is NaN, every table entry past a
    sequence's pages is no page, and the first ``shared`` positions lie in the same pages. The pools are
    one layer of a larger buffer (pages and heads are strided)."""

    def __init__(self, lens, new, Hk, D, page, shared=0, spare=3, seed=0, device="cuda"):
        g = torch.Generator(device="cpu").manual_seed(seed)
        self.host_lens, self.page, self.Hk, self.D = list(lens), page, Hk, D
        self.new = [1] * len(lens) if new is None else list(new)
        common = -(-shared // page) if shared else 0
        own = [max(-(-max(n, 0) // page) - common, 0) for n in lens]
        total = common + sum(own) + spare
        width = max([-(-max(n, 0) // page) for n in lens] + [common, 1]) + 2
        order = torch.randperm(total, generator=g).tolist()
        table = torch.full((len(lens), width + 3), -1, dtype=torch.int32)
        table[:, 1::2] = 1 << 30
        at = common
        for b, n in enumerate(own):
            table[b, :common] = torch.tensor(order[:common], dtype=torch.int32)
            table[b, common:common + n] = torch.tensor(order[at:at + n], dtype=torch.int32)
            at += n
        self.cpu_table = table[:, :width]
        pools = torch.full((2, total, 2, Hk, page + 16, D), NAN, dtype=BF16)
        self.k, self.v = (pools[i, :, 1, :, :page] for i in range(2))
        for b, n in enumerate(lens):
            for j in range(max(n, 0)):
                pg, r = int(table[b, j // page]), j % page
                if j >= shared or torch.isnan(self.k[pg, 0, r, 0]):
                    self.k[pg, :, r] = torch.randn(Hk, D, generator=g).to(BF16)
                    self.v[pg, :, r] = torch.randn(Hk, D, generator=g).to(BF16)
        pools = pools.to(device)
        self.k, self.v = (pools[i, :, 1, :, :page] for i in range(2))
        self.table = table.to(device)[:, :width]
        self.lens = torch.tensor(list(lens), dtype=torch.int32, device=device)
        self.T = sum(self.new)
        self.q_start = None
        if new is not None:
            self.q_start = torch.tensor([0] + list(new)).cumsum(0).to(torch.int32).to(device)

    def rows(self):
        """(token row, sequence, position) of every token."""
        t = 0
        for b, nn in enumerate(self.new):
            for i in range(nn):
                yield t, b, self.host_lens[b] - nn + i
                t += 1

    def gather(self, pool, b, n):
        """Positions 0 .. n - 1 of sequence b [Hk, n, D] in float64 (on the CPU)."""
        pool = pool.cpu()
        ids = self.cpu_table[b, :max(-(-n // self.page), 1)].long().clamp(0, pool.shape[0] - 1)
        return pool[ids].transpose(0, 1).reshape(self.Hk, -1, self.D)[:, :n].double()


def attention(batch, q, Hq, window=0, sinks=0, scale=None, hidden=None):
    """q [T, Hq * D] -> [T, Hq, D] float64; hidden(b, positions): positions left out besides."""
    D, rep = batch.D, Hq // batch.Hk
    scale = D ** -0.5 if scale is None else scale
    q = q.cpu().double().view(-1, Hq, D)
    out = torch.zeros(batch.T, Hq, D, dtype=torch.float64)
    row = 0
    for b, (n, nn) in enumerate(zip(batch.host_lens, batch.new)):
        if n > 0 and nn > 0:
            k, v = batch.gather(batch.k, b, n), batch.gather(batch.v, b, n)
            j = torch.arange(n)
            gone = torch.zeros(n, dtype=torch.bool) if hidden is None else hidden(b, j)
            v = torch.where(gone[:, None], 0.0, v)
            qpos = torch.arange(n - nn, n)[:, None]
            see = (j <= qpos) & ~gone
            if window:
                see &= (j > qpos - window) | (j < sinks)
            v = torch.where(see.any(0)[:, None], v, 0.0)
            for h in range(Hq):
                s = (q[row:row + nn, h] @ k[h // rep].t()) * scale
                s = s.masked_fill(~see, -math.inf)
                m = s.amax(1, keepdim=True)
                p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
                total = p.sum(1, keepdim=True)
                out[row:row + nn, h] = torch.where(total > 0, (p / total) @ v[h // rep], 0.0)
        row += nn
    return out
