"""A batch over a paged cache in 8 bits in plain float64, for the tests of its operators."""
import torch

import paged_ref as R

FP8, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
LEAST, MOST = -110, 119


def exponent(top):
    """The least e with top <= 448 * 2^e, held to the format's limits (top: float64, not negative)."""
    m, e = torch.frexp(top)
    e = e - 9 + (m > 0.875).to(e.dtype)
    return torch.where(top > 0, e, LEAST).clamp(LEAST, MOST)


def strided_codes(codes, device):
    """[n_pages, Hk, page, D] as one layer of a larger buffer (pages and heads strided), what lies between NaN."""
    n, h, p, d = codes.shape
    buf = torch.full((n, 2, h, p + 16, d), 0x7f, dtype=torch.uint8, device=device)
    view = buf[:, 1, :, :p]
    view.copy_(codes.view(torch.uint8))
    return view.view(FP8)


def strided_scales(scales, device):
    n, h, b = scales.shape
    buf = torch.full((n, 2, h, b + 3), 255, dtype=torch.uint8, device=device)
    view = buf[:, 1, :, :b]
    view.copy_(scales.view(torch.uint8))
    return view.view(E8M0)


class Fp8Batch(R.PagedBatch):
    """A PagedBatch whose pools are held in 8 bits (``k8``, ``v8``, ``ks``, ``vs``) and whose ``k`` and ``v`` are the
    values that those stand for. Scales of blocks without a position are 255; ``spread``: blocks differ in magnitude
    by up to 2 to that power."""

    def __init__(self, lens, new, Hk, D, page, spread=4, device="cuda", **kw):
        super().__init__(lens, new, Hk, D, page, device="cpu", **kw)
        g = torch.Generator().manual_seed(kw.get("seed", 0) + 77)
        for name in ("k", "v"):
            x = getattr(self, name).double()
            n = x.shape[0]
            x = x.reshape(n, Hk, page // 16, 16, D)
            live = ~torch.isnan(x)
            # (keys keep their magnitude on the whole, or a few would decide every softmax)
            by = torch.randint(-spread, (spread if name == "v" else 0) + 1, (n, Hk, page // 16, 1, 1), generator=g).double()
            x = torch.where(live, x * torch.exp2(by), 0.0)
            e = exponent(x.abs().amax((3, 4)))
            codes = torch.where(live, (x * torch.exp2(-e.double())[..., None, None]), R.NAN).float().to(FP8)
            some = live.any(4).any(3)
            values = codes.float() * torch.exp2(e.float())[..., None, None]
            scales = torch.where(some, e + 127, 255).to(torch.uint8)
            setattr(self, name, values.reshape(n, Hk, page, D).to(R.BF16).to(device))
            assert torch.equal(getattr(self, name).cpu().float().nan_to_num(1e9), values.reshape(n, Hk, page, D).nan_to_num(1e9))
            setattr(self, name + "8", strided_codes(codes.reshape(n, Hk, page, D), device))
            setattr(self, name + "s", strided_scales(scales, device))
        self.table, self.lens = self.table.to(device), self.lens.to(device)
        if self.q_start is not None:
            self.q_start = self.q_start.to(device)

    def cache(self):
        return self.k8, self.v8, self.ks, self.vs
