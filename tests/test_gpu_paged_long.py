"""Attention over a paged cache of 8 bits, and through a window with first tokens that stay visible, against its formula in 64 bits."""
import math

import pytest
import torch

from helpers import pkg
from paged8_fixtures import LongBatch
from paged_fixtures import held

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32
SHAPES = [(32, 8, 128, 16), (6, 2, 64, 32), (8, 8, 128, 64), (16, 1, 64, 16), (32, 1, 128, 128), (5, 1, 128, 256)]


def check(b, **kw):
    ref, tol = b.expected()
    got = b.run(pkg(), **kw)
    assert pkg().device_status() == 0
    held(got[:ref.shape[0]], ref, tol)
    return got


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
def test_single_tokens_over_codes(dtype, heads, kv_heads, dim, page):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 700, 255, 256, 257]
    check(LongBatch(lens, [1] * len(lens), heads, kv_heads, dim, page, dtype, one_each=True))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(32, 8, 128, 16), (6, 2, 64, 64), (4, 4, 128, 32), (16, 1, 64, 256), (32, 4, 128, 128), (7, 1, 64, 16)])
@pytest.mark.parametrize("new,lens", [([2, 1, 3], [2, 50, 300]), ([9, 8, 17, 1], [9, 8, 150, 1]), ([40, 1, 0, 33], [333, 129, 77, 33]), ([130, 257], [130, 500]), ([64, 128], [64, 1000])])
def test_chunks_over_codes(dtype, heads, kv_heads, dim, page, new, lens):
    check(LongBatch(lens, new, heads, kv_heads, dim, page, dtype, seed=len(lens)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 90]])
def test_blocks_of_very_different_sizes(dtype, new):
    check(LongBatch([400, 90, 1000], new, 8, 2, 128, 32, dtype, spread=30, scatter=2.0 ** -28, seed=3))
    check(LongBatch([400, 90, 1000], new, 8, 2, 64, 32, dtype, spread=6, scatter=2.0 ** -5, seed=4))


@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (7, 0), (16, 4), (64, 64), (100, 5), (130, 129), (333, 17), (2000, 3), (5, 300)])
def test_windows(dtype, codes, window, sinks):
    lens = [1, 5, 16, 40, 129, 200, 257, 640, 1000, 1300]
    check(LongBatch(lens, [1] * len(lens), 32, 8, 128, 16, dtype, codes, window, sinks, one_each=True))
    check(LongBatch(lens, [1, 3, 16, 2, 100, 9, 130, 1, 300, 0], 8, 2, 64, 32, dtype, codes, window, sinks))
    check(LongBatch([700, 2000], [600, 300], 4, 4, 128, 64, dtype, codes, window, sinks, seed=5))


@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_long_rows(dtype, codes):
    check(LongBatch([40000, 3, 9000], [1, 1, 1], 8, 2, 128, 64, dtype, codes, 5000, 4, one_each=True))
    check(LongBatch([9000, 5, 900], [200, 1, 900], 8, 2, 128, 64, dtype, codes, 1024, 4, seed=4))
    check(LongBatch([2100, 5, 900], [600, 1, 900], 8, 2, 128, 64, dtype, codes, 2000 if not codes else 0, 0, seed=4))


@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_hidden_places_hold_anything(dtype, codes, bad):
    """Keys and values ahead of every token's window, NaN or Inf, are not seen.  Not the same bits: where a product of matrices met them the row is computed again key by key, with
    weights that are not rounded, so each result is held to the formula's tolerance, which counts that rounding (2^-8 of the weights over bf16)."""
    for window, sinks, new in ((50, 3, [1, 1]), (50, 0, [40, 20]), (20, 17, [200, 3])):
        b = LongBatch([500, 700], new, 8, 2, 128, 32, dtype, codes, window, sinks, hide=False)
        ref, tol = b.expected()
        held(b.run(pkg()), ref, tol)
        for r, (n, m) in enumerate(zip(b.lens, b.new)):
            for pos in range(sinks, max(0, n - m - window + 1)):
                for pages in (b.k_pages, b.v_pages):
                    pages[b.table[r, pos // 32].item(), :, pos % 32] = torch.full((2, 128), bad if not codes else math.nan).to(pages.dtype).cuda()
        held(b.run(pkg()), ref, tol)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 40])
def test_nan_in_sight_is_seen(dtype, new):
    b = LongBatch([300], [new], 8, 2, 128, 32, dtype, True, 0, 0)
    b.v_pages.view(torch.uint8)[b.table[0, 9].item(), 1, 11] = 0x7f   # position 299: the last token alone sees it
    got = b.run(pkg())
    assert torch.isnan(got[-1, 4:]).all() and torch.isfinite(got[:, :4]).all() and torch.isfinite(got[:-1]).all()


@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_without_tokens_and_queries_without_keys(dtype, codes):
    window, sinks = (0, 0) if codes else (6, 2)
    check(LongBatch([0, 3, 10, 0], [0, 1, 2, 0], 8, 2, 64, 16, dtype, codes, window, sinks))
    b = LongBatch([40], [8], 8, 2, 64, 16, dtype, codes, window, sinks)
    b.lens_dev.fill_(3)
    got = b.run(pkg())
    assert (got[:5] == 0).all() and torch.isfinite(got).all() and (got[5:] != 0).any()
    pkg().device_status()


@pytest.mark.parametrize("codes,window", [(True, 0), (True, 60), (False, 60)])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("max_new", [None, 1, 12, 100])
def test_any_bound_on_new_tokens(dtype, codes, window, max_new):
    check(LongBatch([70, 333, 90], [12, 1, 60], 8, 2, 64, 16, dtype, codes, window, 3 if window else 0), max_new=max_new)


def test_a_window_wider_than_the_row_is_none():
    for codes in (True, False):
        for new in ([1, 1], [30, 200]):
            b = LongBatch([400, 333], new, 8, 2, 128, 32, BF, codes, 401, 0)
            got = b.run(pkg())
            b.window = 0
            assert torch.equal(got, b.run(pkg()))


def test_tables_out_of_bounds_are_reported():
    for window in (0, 40):
        b = LongBatch([100, 90], [1, 30], 8, 2, 128, 16, BF, True, window, 0)
        b.table[1, 5] = 1 << 20
        b.run(pkg())
        assert pkg().device_status() == -7
        assert pkg().device_status() == 0


def test_recorded_call_serves_other_lengths():
    b = LongBatch([900, 500], [1, 1], 8, 2, 128, 32, BF, True, 100, 4, one_each=True, hide=False)
    p = pkg()
    out = torch.empty_like(b.q)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        b.run(p, out=out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            b.run(p, out=out)
        for lens in ([900, 500], [333, 42], [1, 128]):
            b.lens_dev.copy_(torch.tensor(lens, dtype=torch.int32))
            g.replay()
            s.synchronize()
            b.lens = lens
            kept = b.k, b.v
            b.k, b.v = ([x[:n] for x, n in zip(xs, lens)] for xs in kept)
            ref, tol = b.expected()
            held(out, ref, tol)
            b.k, b.v = kept
