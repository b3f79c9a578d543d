"""Plain forms in 64 bits of the operators of a serving step over a paged cache, and batches to try them on."""
import math

import torch

STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half a step of rounding, relative


def rounded_off(ref, dtype):
    """Half a step of a value's rounding to `dtype`: relative to it, and below the smallest normal value half of the subnormals' step, which is
    eps times the smallest normal (f16: 2^-10 2^-14, half of it 2^-25; a value of 1e-5 has a relative half step of only 5e-9)."""
    return torch.clamp(ref.abs() * STEP[dtype] * 1.001, min=torch.finfo(dtype).eps * torch.finfo(dtype).tiny / 2)


def turned(x, positions, f, layout="half", m=1.0):
    """x [tokens, heads, dim] rotated, in f64."""
    n = f.numel()
    x = x.double()
    a = positions.double()[:, None] * f.double()
    c, s = m * a.cos()[:, None], m * a.sin()[:, None]
    out = x.clone()
    i = torch.arange(n, device=x.device)
    first, second = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
    out[..., first] = x[..., first] * c - x[..., second] * s
    out[..., second] = x[..., first] * s + x[..., second] * c
    return out


def turned_off(x, f, dtype, ref, layout="half", m=1.0):
    """How far a rotated tensor may be from `ref`.  cos and sin are off by a unit in the last place (2^-24 at most below 1) and 2^-29
    of an angle's rounding, times m rounded (2^-24): 2^-22.5 with both.  Two products and their sum in f32 round to 2^-24 of each.  Together
    less than 2^-21.5 of |x| + |y|, then half a step of the result's own type.  Dimensions that do not turn are exact."""
    n = f.numel()
    x = x.double().abs()
    i = torch.arange(n, device=x.device)
    first, second = (i, i + n) if layout == "half" else (2 * i, 2 * i + 1)
    tol = torch.zeros_like(x)
    tol[..., first] = tol[..., second] = abs(m) * 2.0 ** -21.5 * (x[..., first] + x[..., second])
    tol[..., :2 * n] += rounded_off(ref, dtype)[..., :2 * n]
    return tol


class Batch:
    """Rows of a paged cache with `lens` tokens, the last `new` of each new; pages lie anywhere, and what no token fills is NaN."""

    def __init__(self, lens, new, heads, kv_heads, dim, page, dtype=torch.bfloat16, seed=0, one_each=False, extra=0, spare=3, device="cuda", fill=math.nan, scatter=1.5):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.new, self.heads, self.kv_heads, self.dim, self.page, self.dtype = list(lens), list(new), heads, kv_heads, dim, page, dtype
        need = [-(-n // page) for n in lens]
        pages, width = sum(need) + spare, max(need + [1]) + 2
        order = torch.randperm(pages, generator=g)
        table = torch.full((len(lens), width), -7, dtype=torch.int32)   # entries that no token needs are never read
        at = 0
        for r, n in enumerate(need):
            table[r, :n] = order[at:at + n].to(torch.int32)
            at += n
        self.k_pages, self.v_pages = (torch.full((pages, kv_heads, page, dim), fill, dtype=dtype, device=device) for _ in range(2))
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.starts_list, self.T = starts, starts[-1] + extra
        self.q = (torch.randn(self.T, heads, dim, generator=g) * scatter).to(dtype).to(device)
        self.k, self.v = ([torch.randn(n, kv_heads, dim, generator=g).to(dtype).to(device) for n in lens] for _ in range(2))
        for r, n in enumerate(lens):
            for j in range(0, n, page):
                m = min(page, n - j)
                self.k_pages[table[r, j // page].item(), :, :m] = self.k[r][j:j + m].transpose(0, 1)
                self.v_pages[table[r, j // page].item(), :, :m] = self.v[r][j:j + m].transpose(0, 1)
        self.table = table.to(device)
        self.lens_dev = torch.tensor(lens, dtype=torch.int32, device=device)
        self.starts = None if one_each else torch.tensor(starts, dtype=torch.int32, device=device)
        self.scale = dim ** -0.5

    def run(self, pkg, max_new=None, out=None):
        return pkg.dispatch.attention_paged(self.q, self.k_pages, self.v_pages, self.table, self.lens_dev, self.scale, self.starts, max_new, out)

    def expected(self):
        """The attention of every new token in f64, and how far a kernel may be from it.  Scores: a product of `dim` terms in f32, off by (dim + 4) 2^-24
        of sum |q k|; a weight by the exponential of twice that (its own score and the maximum's), 2^-22 (the f32 exponent of a score up to 64 in
        powers of two rounds to 2^-19 at most, of those here to 2^-20) and, over bf16, half a step of its own rounding; sums of n terms by (n + 8) 2^-24.  All
        of it relative to sum p |v|, twice because the sum of weights divides; then half a step of the output's type."""
        group = self.heads // self.kv_heads
        refs, tols = [], []
        for r, (n, m) in enumerate(zip(self.lens, self.new)):
            q = self.q[self.starts_list[r]:self.starts_list[r] + m].double()
            k, v = (x[r].double().repeat_interleave(group, dim=1) for x in (self.k, self.v))
            if m == 0 or n == 0:
                refs.append(torch.zeros_like(q)); tols.append(torch.zeros_like(q))
                continue
            s = torch.einsum("ihd,jhd->hij", q, k) * self.scale
            mag = torch.einsum("ihd,jhd->hij", q.abs(), k.abs()) * abs(self.scale)
            late = torch.arange(n, device=q.device)[None, :] > torch.arange(n - m, n, device=q.device)[:, None]
            p = torch.exp(s.masked_fill(late, -math.inf) - s.masked_fill(late, -math.inf).amax(-1, keepdim=True).clamp(min=-1e300))
            p = p.masked_fill(late, 0.0)
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            vz = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
            ref = torch.einsum("hij,jhd->ihd", p, vz)
            spread = torch.einsum("hij,jhd->ihd", p, vz.abs())
            off = 2 * (2 * (self.dim + 4) * 2.0 ** -24 * mag.masked_fill(late, 0.0).amax(-1) + 2.0 ** -20 + (n + 8) * 2.0 ** -24)
            if self.dtype == torch.bfloat16:
                off = off + 2.0 ** -8
            refs.append(ref)
            tols.append(off.transpose(0, 1)[..., None] * spread + ref.abs() * STEP[self.dtype] * 1.01 + 1e-30)
        return torch.cat(refs), torch.cat(tols)


def held(got, ref, tol):
    got = got.double()
    assert torch.isfinite(got).all(), f"{int((~torch.isfinite(got)).sum())} values are not finite"
    worst = ((got - ref).abs() / tol.clamp(min=1e-300)).max().item() if got.numel() else 0.0
    assert worst <= 1.0, f"{worst:.3g} of what is allowed"
