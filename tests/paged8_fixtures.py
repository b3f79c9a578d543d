"""Batches over a paged cache of 8 bits or through a window, and their attention in 64 bits."""
import math

import torch

from paged_fixtures import STEP, Batch

BLOCK = 16


def scales_for(x):
    """Powers of two with which x [..., BLOCK, dim], divided by them, is at most 448."""
    m, e = torch.frexp(x.abs().amax((-1, -2)).double())
    return torch.exp2(torch.where(m > 0, e - 9 + (m > 0.875), torch.full_like(e, -118)).clamp(min=-118).double()).float()


class LongBatch(Batch):
    """A ``Batch`` whose new tokens see their last ``window`` keys (0: all) and the first ``sinks``, over pages of its own type or (``codes``) of 8 bits.  Table entries of
    pages that hold no key in sight are out of the pool."""

    def __init__(self, lens, new, heads, kv_heads, dim, page, dtype=torch.bfloat16, codes=True, window=0, sinks=0, spread=0, hide=True, **kw):
        super().__init__(lens, new, heads, kv_heads, dim, page, dtype, **kw)
        self.window, self.sinks, self.scales = window, sinks, None
        table = self.table.cpu()
        if codes:
            g = torch.Generator().manual_seed(7)
            self.k, self.v = [x.double().cpu() for x in self.k], [x.double().cpu() for x in self.v]
            P, kv, _, d = self.k_pages.shape
            made = []
            for name in ("k", "v"):
                pages = torch.full((P, kv, page, d), math.nan, dtype=torch.float32)    # NaN wherever no token is
                scales = torch.full((P, kv, page // BLOCK), math.nan)
                for r, n in enumerate(lens):
                    x = getattr(self, name)[r]
                    if spread:   # blocks of very different sizes
                        x = x * torch.exp2(torch.randint(-spread, spread + 1, (-(-max(n, 1) // BLOCK), kv, 1), generator=g).double()).repeat_interleave(BLOCK, 0)[:n]
                    for j in range(0, n, BLOCK):
                        m = min(BLOCK, n - j)
                        here = x[j:j + m].transpose(0, 1).float()
                        s = scales_for(here)
                        c = (here / s[:, None, None]).to(torch.float8_e4m3fn)
                        at = table[r, j // page].item()
                        pages[at, :, j % page:j % page + m] = c.float()
                        scales[at, :, j % page // BLOCK] = s
                        x[j:j + m] = (c.double() * s.double()[:, None, None]).transpose(0, 1)
                    getattr(self, name)[r] = x.cuda()
                made.append((pages.to(torch.float8_e4m3fn).cuda(), scales.cuda()))
            (self.k_pages, ks), (self.v_pages, vs) = made
            self.scales = (ks, vs)
        if window and hide:
            for r, (n, m) in enumerate(zip(lens, new)):
                for i in range(-(-n // page)):
                    if i * page >= sinks and (i + 1) * page <= n - m - window + 1:   # behind the sinks, ahead of the first new token's window
                        table[r, i] = -9
            self.table = table.to(self.table.device)

    def run(self, pkg, max_new=None, out=None):
        return pkg.dispatch.attention_paged(self.q, self.k_pages, self.v_pages, self.table, self.lens_dev, self.scale, self.starts, max_new, out, scales=self.scales, window=self.window,
                                            sinks=self.sinks)

    def expected(self):
        """As ``Batch.expected``, but for what hides keys.  Over codes a score is multiplied by three factors more (2^-24 each, beside a product of dim terms), and queries of bf16 as f16
        of a power of two of the row's own lose 2^-39 of its largest element at most; those of chunks, in two e4m3 terms of which the largest
        is at least 224 and the least step 2^-9, lose 2^-10 / 224 < 2^-17.8 of it in each product, twice in a weight and twice in a quotient.  A weight as f16 (2^-11) is within bf16's 2^-8."""
        group = self.heads // self.kv_heads
        refs, tols = [], []
        for r, (n, m) in enumerate(zip(self.lens, self.new)):
            q = self.q[self.starts_list[r]:self.starts_list[r] + m].double()
            if m == 0 or n == 0:
                refs.append(torch.zeros_like(q)); tols.append(torch.zeros_like(q))
                continue
            k, v = (x[r].double().repeat_interleave(group, dim=1) for x in (self.k, self.v))
            i, j = torch.arange(n - m, n, device=q.device)[:, None], torch.arange(n, device=q.device)[None, :]
            hidden = j > i
            if self.window:
                hidden = hidden | ((i - j >= self.window) & (j >= self.sinks))
            kz, vz = (torch.where(torch.isfinite(x), x, torch.zeros_like(x)) for x in (k, v))
            s = (torch.einsum("ihd,jhd->hij", q, kz) * self.scale).masked_fill(hidden, -math.inf)
            mag = torch.einsum("ihd,jhd->hij", q.abs(), kz.abs()) * abs(self.scale) + 2.0 ** -15 * q.abs().amax(-1).T[:, :, None] * kz.abs().sum(-1).T[:, None, :] * abs(self.scale) * (self.scales is not None) * 2.0 ** -8
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)).masked_fill(hidden, 0.0)
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            ref = torch.einsum("hij,jhd->ihd", p, vz)
            spread = torch.einsum("hij,jhd->ihd", p, vz.abs())
            off = 2 * (2 * (self.dim + 8) * 2.0 ** -24 * mag.masked_fill(hidden, 0.0).amax(-1) + 2.0 ** -20 + (n + 8) * 2.0 ** -24)
            if self.dtype == torch.bfloat16:
                off = off + 2.0 ** -8
                if self.scales is not None:
                    lost = 2.0 ** -17.8 * abs(self.scale) * q.abs().amax(-1).T[:, :, None] * kz.abs().sum(-1).T[:, None, :]
                    off = off + 4 * lost.masked_fill(hidden, 0.0).amax(-1)
            refs.append(ref)
            tols.append(off.transpose(0, 1)[..., None] * spread + ref.abs() * STEP[self.dtype] * 1.01 + 1e-30)
        return torch.cat(refs), torch.cat(tols)
