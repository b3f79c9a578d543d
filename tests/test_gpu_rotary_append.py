"""Rotary positions and the append to a paged cache against their formulas in 64 bits."""
import math

import pytest
import torch

from helpers import pkg
from paged_fixtures import Batch, held, turned, turned_off

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def freq(n, base=10000.0, scaling=None):
    return pkg().dispatch.rotary_frequencies(2 * n, base, scaling)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("heads,kv_heads,dim,rot", [(32, 8, 128, 128), (6, 2, 64, 24), (3, 1, 80, 80), (5, 5, 96, 6), (1, 1, 2, 2), (4, 2, 256, 64), (7, 0, 64, 64), (2, 1, 66, 50)])
@pytest.mark.parametrize("tokens", [1, 3, 257])
def test_rotary(dtype, layout, heads, kv_heads, dim, rot, tokens):
    p = pkg()
    g = torch.Generator(device="cuda").manual_seed(tokens)
    q, k = (torch.randn(tokens, h, dim, generator=g, device="cuda").to(dtype) for h in (heads, max(kv_heads, 1)))
    k = k if kv_heads else None
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda", dtype=torch.int64 if tokens == 3 else torch.int32)
    f = freq(rot // 2)
    got = p.dispatch.rotary_apply(q, k, pos, f, layout, 1.1)
    for x, y in ((q, got[0]), (k, got[1])):
        if x is None:
            assert y is None
            continue
        ref = turned(x, pos, f, layout, 1.1)
        held(y, ref, turned_off(x, f, dtype, ref, layout, 1.1))
        assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("pos", [0, 1, 2 ** 31 - 1, -5, 2 ** 40])
def test_rotary_of_positions_far_away(pos):
    """The angle at 2^31 is as good as at 1: f64 frequencies are off by 2^-53 of themselves, the position's product by 2^-22 turns at 2^31."""
    p = pkg()
    q = torch.randn(4, 2, 64, device="cuda")
    at = torch.full((4,), pos, dtype=torch.int64, device="cuda")
    f = freq(32)
    # the angle in whole turns removed exactly, in rational arithmetic on the host
    from fractions import Fraction
    got = p.dispatch.rotary_apply(q, None, at, f, "half")[0]
    two_pi = Fraction("6.283185307179586476925286766559005768394338798750211641949889")
    angles = []
    for v in f.cpu().tolist():
        a = Fraction(v) * pos
        angles.append(float(a - two_pi * (a // two_pi)))
    a = torch.tensor(angles, dtype=torch.float64, device="cuda")
    x, y = q[..., :32].double(), q[..., 32:].double()
    ref = torch.cat([x * a.cos() - y * a.sin(), x * a.sin() + y * a.cos()], -1)
    tol = (x.abs() + y.abs()).repeat(1, 1, 2) * (2.0 ** -21.5 + abs(pos) * 2.0 ** -52) + ref.abs() * 2.0 ** -24
    held(got, ref, tol)


def test_rotary_in_place_from_a_fused_projection():
    p = pkg()
    qkv = torch.randn(37, (6 + 2 + 2) * 64, device="cuda").to(BF)
    q, k = qkv[:, :6 * 64].view(37, 6, 64), qkv[:, 6 * 64:8 * 64].view(37, 2, 64)
    rest, pos, f = qkv[:, 8 * 64:].clone(), torch.arange(37, device="cuda"), freq(32)
    want = p.dispatch.rotary_apply(q.contiguous(), k.contiguous(), pos, f)
    got = p.dispatch.rotary_apply(q, k, pos, f, out=(q, k))
    assert got[0].data_ptr() == qkv.data_ptr()
    assert torch.equal(q, want[0]) and torch.equal(k, want[1]) and torch.equal(qkv[:, 8 * 64:], rest)


def test_rotary_matches_the_unscaled_half_rotation_of_the_decoder():
    p = pkg()
    x = torch.randn(1, 50, 4, 64, device="cuda")
    cos, sin = p.dispatch.rotation_tables(64, 64, 10000.0)
    old = p.dispatch.fused_rope_apply(x, cos, sin, 3)[0]
    new = p.dispatch.rotary_apply(x[0], None, torch.arange(3, 53, device="cuda"), freq(32))[0]
    pairs = (x[0][..., :32].abs() + x[0][..., 32:].abs()).repeat(1, 1, 2)
    assert ((old - new).abs() <= pairs * 2.0 ** -20).all()   # both are within 2^-21.5 of the formula


def test_scaled_frequencies():
    p = pkg()
    d = p.dispatch
    f = d.rotary_frequencies(64, 10000.0, None, "cpu")
    assert torch.equal(d.rotary_frequencies(64, 10000.0, d.RotaryScaling("linear", 4.0), "cpu"), f / 4)
    b = d.rotary_frequencies(64, 10000.0, d.RotaryScaling("base", 4.0), "cpu")
    assert abs(b[0].item() - 1) < 1e-12 and abs(b[-1].item() / (f[-1].item() / 4) - 1) < 1e-9
    s = d.RotaryScaling("ramp", 4.0, original=2048)
    r = d.rotary_frequencies(64, 10000.0, s, "cpu")
    turns = 2048 * f / (2 * math.pi)
    assert torch.equal(r[turns >= 32], f[turns >= 32]) and torch.equal(r[turns <= 1], f[turns <= 1] / 4)
    assert ((r <= f) & (r >= f / 4)).all() and abs(s.magnitude - (0.1 * math.log(4) + 1)) < 1e-12
    for bad in (d.RotaryScaling("other", 2.0), d.RotaryScaling("linear", 0.0), d.RotaryScaling("ramp", 2.0)):
        with pytest.raises(p.Ab2Error):
            d.rotary_frequencies(64, 10000.0, bad, "cpu")


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot,page", [(128, 128, 16), (64, 64, 32), (64, 24, 128), (128, 0, 64), (64, 6, 256)])
@pytest.mark.parametrize("lens,new", [([1, 17, 300], [1, 1, 1]), ([5, 130, 0, 33, 64], [5, 67, 0, 1, 64])])
def test_append(dtype, layout, dim, rot, page, lens, new):
    p = pkg()
    b = Batch(lens, new, 6, 2, dim, page, dtype, one_each=max(new) == 1, extra=0 if max(new) == 1 else 3, seed=dim)
    n = b.starts_list[-1]
    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn(b.T, 2, dim, generator=g, device="cuda").to(dtype) for _ in range(2))
    f = freq(rot // 2) if rot else None
    want_k, want_v = b.k_pages.clone(), b.v_pages.clone()
    pos = torch.cat([torch.arange(L - m, L) for L, m in zip(lens, new)]).cuda()
    row = torch.cat([torch.full((m,), r) for r, m in enumerate(new)]).cuda()
    where, slot = b.table[row, pos // page].long(), pos % page
    fd = f if rot else torch.zeros(0, dtype=torch.float64, device="cuda")
    ref_k, ref_q = (turned(x[:n], pos, fd, layout, 0.9) for x in (k, b.q))
    out = torch.full((b.T, 6, dim), 3.0, dtype=dtype, device="cuda")
    got = p.dispatch.paged_append(b.k_pages, b.v_pages, k, v, b.table, b.lens_dev, b.starts, q=b.q, frequencies=f, layout=layout, magnitude=0.9, out=out)
    assert p.device_status() == 0 and got is out
    held(b.k_pages[where, :, slot], ref_k, turned_off(k[:n], fd, dtype, ref_k, layout, 0.9))
    held(got[:n], ref_q, turned_off(b.q[:n], fd, dtype, ref_q, layout, 0.9))
    assert (out[n:] == 3).all()
    assert torch.equal(b.v_pages[where, :, slot], v[:n])
    for pool, old in ((b.k_pages, want_k), (b.v_pages, want_v)):   # and nothing else
        old[where, :, slot] = pool[where, :, slot]
        assert torch.equal(torch.nan_to_num(pool.float(), nan=-99.0), torch.nan_to_num(old.float(), nan=-99.0))


def test_append_without_queries_from_strided_rows_and_many_rows():
    p = pkg()
    lens = [1 + r % 40 for r in range(100)]
    b = Batch(lens, [1 + r % 3 if L > 3 else 1 for r, L in enumerate(lens)], 4, 2, 64, 16, BF, fill=0.0)
    n = b.starts_list[-1]
    kv = torch.randn(n, 4, 64, device="cuda").to(BF)
    k, v = kv[:, :2], kv[:, 2:]
    assert p.dispatch.paged_append(b.k_pages, b.v_pages, k, v, b.table, b.lens_dev, b.starts) is None
    pos = torch.cat([torch.arange(L - m, L) for L, m in zip(lens, b.new)]).cuda()
    row = torch.cat([torch.full((m,), r) for r, m in enumerate(b.new)]).cuda()
    where = b.table[row, pos // 16].long()
    assert torch.equal(b.k_pages[where, :, pos % 16], k) and torch.equal(b.v_pages[where, :, pos % 16], v)
    assert p.device_status() == 0


def test_append_to_bad_places_writes_nothing_there():
    p = pkg()
    b = Batch([40, 20], [3, 2], 4, 2, 64, 16, BF, fill=0.0)
    k, v = (torch.randn(5, 2, 64, device="cuda").to(BF) for _ in range(2))
    before = b.k_pages.clone(), b.v_pages.clone()
    keep = b.table.clone()
    b.table[0] = 10 ** 7
    b.table[1] = -2
    p.dispatch.paged_append(b.k_pages, b.v_pages, k, v, b.table, b.lens_dev, b.starts, q=b.q, frequencies=freq(32))
    assert p.device_status() == -7
    b.table.copy_(keep)
    b.lens_dev.copy_(torch.tensor([2, 0], dtype=torch.int32))   # shorter than their new tokens
    k0 = b.k_pages.clone()
    assert torch.equal(k0, before[0]) and torch.equal(b.v_pages, before[1])
    p.dispatch.paged_append(b.k_pages, b.v_pages, k, v, b.table, b.lens_dev, b.starts)
    assert p.device_status() == -7
    page = b.table[0, 0].item()
    assert torch.equal(b.k_pages[page, :, :2], k[1:3].transpose(0, 1))   # the two that have places
    k0[page, :, :2] = b.k_pages[page, :, :2]
    assert torch.equal(b.k_pages, k0)


def test_refusals():
    p = pkg()
    d = p.dispatch
    q, k, pos, f = torch.zeros(3, 4, 64, device="cuda"), torch.zeros(3, 2, 64, device="cuda"), torch.arange(3, device="cuda"), freq(32)
    for args in ((q.cpu(), k, pos, f), (q, k[:2], pos, f), (q, k[..., :32], pos, f), (q, k.half(), pos, f), (q, k, pos.float(), f), (q, k, pos[:2], f),
                 (q, k, pos, f.float()), (q, k, pos, freq(33)), (q[0], None, pos, f), (q.double(), None, pos, f), (q, k, pos, f, "other"),
                 (q[..., :63], None, pos, freq(31)), (q, k, pos, f, "half", 1.0, (q.half(), k))):
        with pytest.raises(p.Ab2Error):
            d.rotary_apply(*args)
    assert d.rotary_apply(q[:0], k[:0], pos[:0], f)[0].shape == (0, 4, 64)
    b = Batch([40, 20], [3, 2], 4, 2, 64, 16, BF)
    kk = torch.zeros(5, 2, 64, dtype=BF, device="cuda")
    ok = dict(k_pages=b.k_pages, v_pages=b.v_pages, k=kk, v=kk, table=b.table, lens=b.lens_dev, starts=b.starts, q=b.q, frequencies=f)
    d.paged_append(**ok)
    for bad in (dict(k=kk.float(), v=kk.float()), dict(v=kk[:3]), dict(k=kk[:, :1], v=kk[:, :1]), dict(q=b.q[:2]), dict(q=b.q.float()), dict(starts=None), dict(frequencies=freq(40)),
                dict(lens=b.lens_dev.long()), dict(table=b.table.cpu()), dict(out=b.q[:1]), dict(layout="no")):
        with pytest.raises(p.Ab2Error):
            d.paged_append(**{**ok, **bad})
