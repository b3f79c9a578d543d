"""The append of keys and values to pages of 8 bits against its formula in 64 bits, and steps over such a cache."""
import math

import pytest
import torch

from helpers import pkg
from paged_fixtures import STEP, held, turned, turned_off

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
BLOCK = 16


def power(amax):
    m, e = torch.frexp(amax.double())
    return torch.exp2(torch.where(m > 0, e - 9 + (m > 0.875), torch.full_like(e, -118)).clamp(min=-118).double())


class Pool:
    """Pages with what earlier tokens left, rows of them, and new tokens."""

    def __init__(self, before, new, heads, kv_heads, dim, page, dtype, seed=0, extra=0, loud=1.0):
        g = torch.Generator().manual_seed(seed)
        self.before, self.new, self.kv, self.dim, self.page, self.dtype = before, new, kv_heads, dim, page, dtype
        lens = [b + n for b, n in zip(before, new)]
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=g)
        self.table = torch.full((len(new), max(need + [1]) + 1), -5, dtype=torch.int32)
        at = 0
        for r, n in enumerate(need):
            self.table[r, :n] = order[at:at + n].int()
            at += n
        self.codes = [(torch.randn(pages, kv_heads, page, dim, generator=g) * 100).clamp(-448, 448).to(torch.float8_e4m3fn) for _ in range(2)]
        self.scales = [torch.exp2(torch.randint(-9, -3, (pages, kv_heads, page // BLOCK), generator=g).float()) for _ in range(2)]
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.starts, self.T = starts, starts[-1] + extra
        self.q = torch.randn(self.T, heads, dim, generator=g).to(dtype).cuda()
        self.x = [(torch.randn(self.T, kv_heads, dim, generator=g) * loud).to(dtype).cuda() for _ in range(2)]
        self.lens = torch.tensor(lens, dtype=torch.int32).cuda()
        self.k_pages, self.v_pages = (c.cuda().clone() for c in self.codes)
        self.ks, self.vs = (s.cuda().clone() for s in self.scales)

    def run(self, f, layout="half", m=1.0, one_each=False, q=True, k=None, v=None):
        starts = None if one_each else torch.tensor(self.starts, dtype=torch.int32).cuda()
        return pkg().dispatch.paged_append(self.k_pages, self.v_pages, self.x[0] if k is None else k, self.x[1] if v is None else v, self.table.cuda(), self.lens, starts,
                                           self.q if q else None, f, layout, m, scales=(self.ks, self.vs))

    def check(self, f, layout, m):
        for kind, (pages, scales) in enumerate(((self.k_pages, self.ks), (self.v_pages, self.vs))):
            got, got_scales = pages.cpu().float().double(), scales.cpu().double()
            was, was_scales = self.codes[kind].float().double(), self.scales[kind].double()
            touched, blocks = torch.zeros(got.shape, dtype=torch.bool), torch.zeros(got_scales.shape, dtype=torch.bool)
            for r, (b, n) in enumerate(zip(self.before, self.new)):
                x = self.x[kind][self.starts[r]:self.starts[r] + n]
                pos = torch.arange(b, b + n, device="cuda")
                exact = turned(x, pos, f, layout, m) if kind == 0 and f is not None else x.double()
                off = turned_off(x, f, self.dtype, exact, layout, m) if kind == 0 and f is not None else torch.zeros_like(exact)   # the rotation and its rounding to the type
                exact, off = exact.cpu(), off.cpu()
                for block in range(b // BLOCK, -(-(b + n) // BLOCK) if n else 0):
                    lo, hi = max(b, block * BLOCK), min(b + n, block * BLOCK + BLOCK)
                    page, at = self.table[r, block * BLOCK // self.page].item(), block * BLOCK % self.page
                    y, e = exact[lo - b:hi - b].transpose(0, 1), off[lo - b:hi - b].transpose(0, 1)
                    fine = y.isfinite()
                    size, slack = torch.where(fine, y, 0.0).abs().amax((1, 2)), torch.where(fine, e, 0.0).amax((1, 2))
                    old = was_scales[page, :, at // BLOCK] if lo > block * BLOCK else torch.zeros(self.kv, dtype=torch.float64)
                    least, most = (torch.maximum(power((size + d).clamp(min=0)), old) for d in (-slack, slack))
                    s = got_scales[page, :, at // BLOCK]
                    assert ((s >= least) & (s <= most)).all()
                    new = got[page, :, at + lo % BLOCK:at + lo % BLOCK + hi - lo]
                    assert torch.equal(new.isnan(), ~fine)
                    u = s[:, None, None]
                    step = torch.maximum(y.abs() / u * 2.0 ** -4, torch.tensor(2.0 ** -10, dtype=torch.float64)) * u    # half a step of e4m3, whose least is 2^-9
                    z = torch.zeros_like(y)
                    held(torch.where(fine, new * u, z), torch.where(fine, y, z), torch.where(fine, step * 1.001 + e * 1.07, z + 1))
                    if lo > block * BLOCK:   # earlier tokens: their values, rounded once more where the scale grew
                        value = was[page, :, at:at + lo % BLOCK] * old[:, None, None]
                        here = got[page, :, at:at + lo % BLOCK] * u
                        exactly = value.abs() >= 2.0 ** -6 * u
                        assert torch.equal(here[exactly], value[exactly])
                        assert ((here - value).abs() <= u * 2.0 ** -10).all()
                    touched[page, :, at:at + lo % BLOCK + hi - lo] = True
                    blocks[page, :, at // BLOCK] = True
            assert torch.equal(got[~touched], was[~touched]) and torch.equal(got_scales[~blocks], was_scales[~blocks])
        assert pkg().device_status() == 0


def freq(n):
    return pkg().dispatch.rotary_frequencies(2 * n) if n else None


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("heads,kv_heads,dim,rot,page", [(32, 8, 128, 128, 16), (6, 2, 64, 24, 64), (16, 4, 128, 64, 32), (5, 1, 64, 6, 16), (3, 3, 128, 0, 256), (4, 2, 64, 64, 128)])
def test_append(dtype, layout, heads, kv_heads, dim, rot, page):
    for before, new in (([0, 5, 16, 31, 700, 15], [1] * 6), ([0, 3, 16, 90, 0, 33], [40, 13, 1, 0, 300, 15]), ([1], [1])):
        p = Pool(before, new, heads, kv_heads, dim, page, dtype, seed=rot + page, loud=3.0)
        f = freq(rot // 2)
        got = p.run(f, layout, 1.25, one_each=all(n == 1 for n in new))
        p.check(f, layout, 1.25)
        if f is not None:
            pos = torch.cat([torch.arange(b, b + n, device="cuda") for b, n in zip(before, new)])
            ref = turned(p.q, pos, f, layout, 1.25)
            held(got, ref, turned_off(p.q, f, dtype, ref, layout, 1.25))
        else:
            assert torch.equal(got, p.q)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_blocks_that_grow_and_blocks_that_do_not(dtype):
    for loud in (1e-3, 1.0, 300.0, 1e6, 1e-30, 1e30):
        p = Pool([7, 40, 0, 16], [1, 20, 3, 16], 4, 2, 128, 32, dtype, seed=3, loud=loud)
        p.run(freq(64))
        p.check(freq(64), "half", 1.0)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_zeros_and_values_that_are_not_finite(dtype):
    p = Pool([0, 3, 0], [16, 9, 4], 4, 2, 64, 16, dtype)
    p.x[1][:16] = 0.0                                    # a block of zeros
    p.x[1][18, 0, 5], p.x[1][20, 1, 7], p.x[1][26] = math.inf, math.nan, -math.inf
    p.run(freq(32))
    p.check(freq(32), "half", 1.0)
    assert (p.v_pages.float().cpu()[p.table[0, 0].item()] == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
def test_parts_of_a_fused_projection(dtype):
    p = Pool([5, 90, 0], [30, 1, 17], 8, 2, 64, 16, dtype, extra=3)
    f = freq(32)
    for shift in (0, 1):   # an odd offset: elements one by one
        fused = torch.zeros(p.T, 12 * 64 + 3 + shift, dtype=dtype, device="cuda")
        parts = [fused[:, shift + a * 64:shift + b * 64].unflatten(1, (-1, 64)) for a, b in ((0, 8), (8, 10), (10, 12))]
        for part, x in zip(parts, (p.q, *p.x)):
            part.copy_(x)
        pages = p.k_pages, p.v_pages, p.ks, p.vs
        p.k_pages, p.v_pages = (c.cuda().clone() for c in p.codes)
        p.ks, p.vs = (s.cuda().clone() for s in p.scales)
        starts = torch.tensor(p.starts, dtype=torch.int32).cuda()
        got = pkg().dispatch.paged_append(p.k_pages, p.v_pages, parts[1], parts[2], p.table.cuda(), p.lens, starts, parts[0], f, "half", 1.0, scales=(p.ks, p.vs))
        p.check(f, "half", 1.0)
        if shift:
            assert torch.equal(got[:-3], first[:-3]) and all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(pages, (p.k_pages, p.v_pages, p.ks, p.vs)))
        first = got


def test_tokens_behind_the_last_row_and_in_place():
    p = Pool([5, 9], [3, 20], 8, 2, 128, 16, BF, extra=4)
    f, q = freq(64), p.q.clone()
    starts = torch.tensor(p.starts, dtype=torch.int32).cuda()
    got = pkg().dispatch.paged_append(p.k_pages, p.v_pages, *p.x, p.table.cuda(), p.lens, starts, p.q, f, out=p.q, scales=(p.ks, p.vs))
    assert got is p.q and torch.equal(p.q[-4:], q[-4:])
    p.check(f, "half", 1.0)
    ref = turned(q[:23], torch.cat([torch.arange(5, 8), torch.arange(9, 29)]).cuda(), f)
    held(got[:23], ref, turned_off(q[:23], f, BF, ref))


def test_what_is_out_of_bounds_is_reported_and_touches_nothing():
    p = Pool([5, 9], [3, 20], 8, 2, 128, 16, BF)
    f = freq(64)
    p.table[1] = 1 << 20
    p.run(f)
    assert pkg().device_status() == -7
    p.table[1] = p.table[0]
    before = p.k_pages.clone(), p.ks.clone()
    p.starts = [0, 40, 20]   # falls, and passes the tokens
    p.lens[:] = 0
    p.run(f)
    assert pkg().device_status() == -7
    assert torch.equal(p.k_pages.view(torch.uint8), before[0].view(torch.uint8)) and torch.equal(p.ks, before[1])
    assert pkg().device_status() == 0


def test_many_rows():
    g = torch.Generator().manual_seed(1)
    for rows in (31, 33, 130, 700):
        before = torch.randint(0, 60, (rows,), generator=g).tolist()
        new = torch.randint(0, 5, (rows,), generator=g).tolist()
        p = Pool(before, new, 2, 1, 64, 16, BF, seed=rows)
        p.run(freq(32))
        p.check(freq(32), "half", 1.0)


def test_a_block_that_grew_token_by_token():
    """It holds what one append of all tokens makes, but for what falls below the least step of a scale on the way."""
    p = pkg()
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v, q = (torch.randn(100, h, 64, generator=g, device="cuda").to(BF) for h in (2, 2, 4))
    k *= torch.logspace(-2, 2, 100, device="cuda").to(BF)[:, None, None]
    f = freq(32)
    caches = [p.PagedKVCache(20, 16, 2, 64, batch=1, dtype="e4m3") for _ in range(2)]
    step = caches[0].step([0], [100])
    caches[0].append(step, k, v, 0, q, f)
    caches[0].commit(step)
    for t in range(100):
        step = caches[1].step([0], [1])
        caches[1].append(step, k[t:t + 1], v[t:t + 1], 0, q[t:t + 1], f)
        caches[1].commit(step)
    (ka, va), (kb, vb) = caches[0].read(), caches[1].read()
    assert torch.equal(caches[0].k_scales, caches[1].k_scales) and torch.equal(va, vb)
    at = torch.arange(100) // 16
    s = caches[0].k_scales[0, torch.tensor(caches[0]._pages[0], device="cuda"), :, 0][at.cuda()]
    # a code is off by up to 2^-10 of every scale on the way, each of which is at most the last: halves of it, quarters, ...
    assert ((ka - kb).abs() <= s[..., None] * 2.0 ** -9).all()
    assert (ka == kb).float().mean() > 0.9


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("window,sinks", [(0, 0), (40, 4)])
def test_steps_of_a_cache(dtype, window, sinks):
    """Prompts in portions, then token by token, appended and attended to as a user's program does: each step against the formula over what the cache holds."""
    p = pkg()
    g = torch.Generator(device="cuda").manual_seed(9)
    cache = p.PagedKVCache(60, 16, 2, 128, batch=3, n_layers=2, dtype="e4m3")
    f = freq(64)
    for rows, new in (([0, 2], [50, 7]), ([1, 0], [3, 33]), ([0, 1, 2], [1, 1, 1]), ([2, 0, 1], [1, 1, 60]), ([0, 1, 2], [1, 1, 1])):
        step = cache.step(rows, new)
        T = sum(new)
        outs = []
        for layer in range(2):
            q, k, v = (torch.randn(T, h, 128, generator=g, device="cuda").to(dtype) for h in (8, 2, 2))
            turned_q = cache.append(step, k, v, layer, q, f)
            outs.append((turned_q, cache.attention(step, turned_q, 0.09, layer, window=window, sinks=sinks)))
        cache.commit(step)
        for layer, (q, o) in enumerate(outs):
            at = 0
            for r, n in zip(rows, new):
                k, v = (x.double().repeat_interleave(4, 1) for x in cache.read(r, layer))
                L = k.shape[0]
                i, j = torch.arange(L - n, L, device="cuda")[:, None], torch.arange(L, device="cuda")[None, :]
                hidden = j > i
                if window:
                    hidden = hidden | ((i - j >= window) & (j >= sinks))
                s = torch.einsum("ihd,jhd->hij", q[at:at + n].double(), k) * 0.09
                w = torch.softmax(s.masked_fill(hidden, -math.inf), -1)
                ref, spread = torch.einsum("hij,jhd->ihd", w, v), torch.einsum("hij,jhd->ihd", w, v.abs())
                # scores of up to 30 in sum |q k| off by 136 2^-24 of that, twice in a weight and twice in a quotient; the weights' own rounding; the output's
                held(o[at:at + n], ref, spread * (4 * 136 * 30 * 2.0 ** -24 + 2.0 ** -19 + (2.0 ** -8 if dtype == BF else 0)) + ref.abs() * STEP[dtype] * 1.01)
                at += n
    assert p.device_status() == 0
