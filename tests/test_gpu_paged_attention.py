"""Attention over a paged cache against its formula in 64 bits."""
import ctypes as C
import math

import pytest
import torch

from helpers import pkg
from paged_fixtures import Batch, held

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def check(b, **kw):
    ref, tol = b.expected()
    got = b.run(pkg(), **kw)
    held(got[:ref.shape[0]], ref, tol)
    assert pkg().device_status() == 0
    return got


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(32, 8, 128, 16), (6, 2, 64, 32), (8, 8, 128, 64), (16, 1, 64, 16), (32, 1, 128, 128), (5, 1, 128, 256)])
def test_single_tokens(dtype, heads, kv_heads, dim, page):
    lens = [1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 128, 129, 700, 255, 256, 257]
    check(Batch(lens, [1] * len(lens), heads, kv_heads, dim, page, dtype, one_each=True))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(32, 8, 128, 16), (6, 2, 64, 64), (4, 4, 128, 32), (16, 1, 64, 256), (32, 4, 128, 128), (7, 1, 64, 16)])
@pytest.mark.parametrize("new,lens", [([2, 1, 3], [2, 50, 300]), ([9, 8, 17, 1], [9, 8, 150, 1]), ([40, 1, 0, 33], [333, 129, 77, 33]), ([130, 257], [130, 500]), ([64, 128], [64, 1000])])
def test_chunks(dtype, heads, kv_heads, dim, page, new, lens):
    check(Batch(lens, new, heads, kv_heads, dim, page, dtype, seed=len(lens)))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,ctx", [(1, 5000), (3, 3001), (40, 300), (200, 100), (700, 20)])
def test_rows_of_many_lengths(dtype, rows, ctx):
    lens = [max(1, ctx * (1 + 7 * r % 11) // 11) for r in range(rows)]
    check(Batch(lens, [1] * rows, 8, 2, 64 if dtype == F32 else 128, 16, dtype, one_each=True, seed=rows))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_long_chunk_behind_a_long_context(dtype):
    check(Batch([2100, 5, 900], [600, 1, 900], 8, 2, 128, 64, dtype, seed=4))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_without_tokens_and_queries_without_keys(dtype):
    b = Batch([0, 3, 10, 0], [0, 1, 2, 0], 8, 2, 64, 16, dtype)
    check(b)
    # more new tokens than tokens: the first ones see nothing and answer zeros
    b = Batch([40], [8], 8, 2, 64, 16, dtype)
    b.lens_dev.fill_(3)
    got = b.run(pkg())
    assert pkg().device_status() == 0
    assert (got[:5] == 0).all() and torch.isfinite(got).all() and (got[5:] != 0).any()
    wide = Batch([300, 70], [300, 70], 8, 2, 64, 16, dtype, seed=1)   # many tiles of queries without keys, one after the other
    wide.lens_dev.copy_(torch.tensor([0, 4], dtype=torch.int32))
    for bound in (300, 1):
        out = wide.run(pkg(), max_new=bound)
        assert pkg().device_status() == 0 and (out[:366] == 0).all() and (out[366:] != 0).any()
    c = Batch([40], [3], 8, 2, 64, 16, dtype)
    c.q, c.k_pages, c.v_pages, c.table = b.q[5:].contiguous(), b.k_pages, b.v_pages, b.table
    c.lens_dev.fill_(3)
    c.lens, c.k, c.v = [3], [b.k[0][:3]], [b.v[0][:3]]
    ref, tol = c.expected()   # the others are the first three tokens' row
    held(got[5:], ref, tol)
    held(c.run(pkg()), ref, tol)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new,heads", [(1, 4), (5, 4), (100, 4), (300, 4)])
def test_what_lies_out_of_sight_does_not_matter(dtype, new, heads):
    """Later keys and values of the same chunk that are Inf or NaN reach only the tokens that see them (what no token fills is NaN in every batch)."""
    b = Batch([200 + new], [new], heads, 1, 128, 32, dtype, seed=9)
    clean = b.run(pkg())
    last = 200 + new - 1
    page, slot = b.table[0, last // 32].item(), last % 32
    for bad_k, bad_v in ((math.nan, math.nan), (1.0, math.inf), (math.inf, 1.0), (torch.finfo(dtype).min, -math.inf)):
        b.k_pages[page, :, slot], b.v_pages[page, :, slot] = bad_k, bad_v
        got = b.run(pkg())
        if new > 1:
            ref, tol = b.expected()
            held(got[:new - 1], ref[:new - 1], tol[:new - 1])
        assert torch.isfinite(clean).all()
    assert not torch.isfinite(got[-1]).all()   # the last token sees it


@pytest.mark.parametrize("dtype", [BF, F32])
def test_scores_far_apart(dtype):
    b = Batch([700, 333], [1, 20], 8, 2, 128, 16, dtype, scatter=30.0)
    ref, _ = b.expected()
    got = b.run(pkg()).double()
    assert torch.isfinite(got).all()
    # nearly all weight on one key: its value, to the output's rounding and the weight of the rest
    assert ((got - ref).abs().max() / ref.abs().max()).item() < (2.0 ** -6 if dtype == BF else 1e-4)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 4, 70])
@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
def test_any_scale(dtype, new, scale):
    b = Batch([300, 95], [new, new], 8, 2, 64, 16, dtype, seed=3, scatter=0.5)
    b.scale = scale
    check(b)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 6, 90])
def test_strides_padding_and_results_in_place(dtype, new):
    p = pkg()
    b = Batch([300, 77], [new, new], 8, 2, 64, 16, dtype, seed=2, extra=5)
    plain = b.run(p)
    n = b.starts_list[-1]
    wide = torch.full((b.T, 8 + 4, 64), math.nan, dtype=dtype, device="cuda")   # q of a fused projection
    wide[:, :8] = b.q
    b.q = wide[:, :8]
    out = torch.full((b.T, 10, 64), 7.0, dtype=dtype, device="cuda")
    got = b.run(p, out=out[:, 1:9])
    assert got.data_ptr() == out[:, 1:9].data_ptr()
    assert torch.equal(got[:n], plain[:n])
    assert (out[:, 0] == 7).all() and (out[:, 9] == 7).all() and (out[n:] == 7).all()   # nothing else is written
    table = torch.full((2, b.table.shape[1] + 9), 10 ** 9, dtype=torch.int32, device="cuda")
    table[:, :b.table.shape[1]] = b.table
    b.table = table[:, :b.table.shape[1]]
    assert torch.equal(b.run(p)[:n], plain[:n])
    # without a 16-byte boundary
    flat = torch.empty(b.T * 8 * 64 + 1, dtype=dtype, device="cuda")
    flat[1:] = b.q.reshape(-1)
    b.q = flat[1:].view(b.T, 8, 64)
    assert torch.equal(b.run(p)[:n], plain[:n])


@pytest.mark.parametrize("dtype", [BF, F32])
def test_without_a_workspace_and_with_any_bound_on_new_tokens(dtype):
    p = pkg()
    for new, lens in (([1, 1], [900, 40]), ([30, 1], [2000, 70]), ([200, 3], [1200, 333])):
        b = Batch(lens, new, 8, 2, 128, 32, dtype, seed=5)
        ref, tol = b.expected()
        for bound in (1, max(new), 10 ** 6, 2 ** 40):
            held(b.run(p, max_new=bound), ref, tol)
        c, keep = p.dispatch._paged(b.k_pages, b.v_pages, b.table, b.lens_dev, b.starts, b.T)
        out = torch.empty_like(b.q)
        p.check(p.lib.ab2_paged_attention(C.byref(c), b.q.data_ptr(), 8 * 128, 8, out.data_ptr(), 8 * 128, max(new), b.scale, None, 0, p.dispatch.dtype_code(dtype), torch.cuda.current_stream().cuda_stream))
        held(out, ref, tol)
    assert p.device_status() == 0


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 4, 150])
def test_the_same_bits_every_time_and_from_two_streams(dtype, new):
    p = pkg()
    a, b = (Batch([1500, 300, 5 + new], [new] * 3, 16, 4, 128, 16, dtype, seed=s) for s in (1, 2))
    want = [a.run(p).clone(), b.run(p).clone()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(10):
        got = []
        for s, x in zip(streams, (a, b)):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                got.append(x.run(p))
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 40])
def test_recorded_calls_follow_the_lengths(dtype, new):
    p = pkg()
    batches = [Batch(lens, [new] * 3, 8, 2, 64, 16, dtype, seed=s, spare=60) for s, lens in ((3, [900, 400, 50 + new]), (4, [300, 20 + new, 40 + new]))]
    pages, width = max(x.k_pages.shape[0] for x in batches), max(x.table.shape[1] for x in batches)
    k, v = (torch.zeros((pages, 2, 16, 64), dtype=dtype, device="cuda") for _ in range(2))
    table, lens, q = torch.zeros((3, width), dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"), torch.zeros_like(batches[0].q)
    out, graphs, stream = [torch.empty_like(q) for _ in range(2)], [], torch.cuda.Stream()
    for o in out:   # two graphs of the same call, replayed one behind the other
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            p.dispatch.attention_paged(q, k, v, table, lens, batches[0].scale, batches[0].starts, new, o)
        graphs.append(g)
    for x in batches + batches[:1]:
        k[:x.k_pages.shape[0]], v[:x.v_pages.shape[0]], table[:, :x.table.shape[1]] = x.k_pages, x.v_pages, x.table
        lens.copy_(x.lens_dev)
        q.copy_(x.q)
        for o, g in zip(out, graphs):
            o.fill_(math.nan)
            g.replay()
        torch.cuda.synchronize()
        ref, tol = x.expected()
        for o in out:
            held(o, ref, tol)
    assert p.device_status() == 0


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [1, 50])
def test_bad_tables_and_lengths_are_reported(dtype, new):
    """What is out of bounds in device memory is brought within them and shows in the status word; the other rows are answered."""
    p = pkg()
    b = Batch([200, 150, 90], [new] * 3, 8, 2, 64, 16, dtype, seed=6, fill=0.0)
    ref, tol = b.expected()
    for page in (10 ** 6, -1, b.k_pages.shape[0]):
        keep = b.table.clone()
        b.table[1, 2] = page
        got = b.run(p)
        assert p.device_status() == -7
        held(torch.cat([got[:new], got[2 * new:]]), torch.cat([ref[:new], ref[2 * new:]]), torch.cat([tol[:new], tol[2 * new:]]))
        b.table.copy_(keep)
    b.lens_dev[2] = 10 ** 9
    keep = b.table.clone()
    b.table.clamp_(min=0)
    got = b.run(p)
    assert p.device_status() == -7
    held(got[:2 * new], ref[:2 * new], tol[:2 * new])
    b.lens_dev[2] = -5
    b.run(p)
    assert p.device_status() == -7
    b.lens_dev[2] = 90
    for bad in ([0, new, new - 1, 2 * new], [0, new, 2 * new, 10 ** 6], [-3, new, 2 * new, 3 * new]):
        b.starts = torch.tensor(bad, dtype=torch.int32, device="cuda")
        b.run(p)
        assert p.device_status() == -7
    b.starts, b.table = torch.tensor([0, new, 2 * new, 3 * new], dtype=torch.int32, device="cuda"), keep
    held(b.run(p), ref, tol)
    assert p.device_status() == 0


def test_pages_past_32_bits():
    """A pool of more than 2^32 elements, the batch's pages at its end."""
    p = pkg()
    pages = (1 << 32) // (2 * 256 * 128) + 40
    b = Batch([600, 300], [1, 20], 8, 2, 128, 256, BF, seed=8, fill=0.0)
    ref, tol = b.expected()
    n = b.k_pages.shape[0]
    k, v = (torch.empty((pages, 2, 256, 128), dtype=BF, device="cuda") for _ in range(2))
    k[-n:], v[-n:] = b.k_pages, b.v_pages
    b.k_pages, b.v_pages, b.table = k, v, torch.where(b.table >= 0, b.table + (pages - n), b.table)
    held(b.run(p), ref, tol)
    got = p.dispatch.paged_append(k, v, b.k[1][-20:], b.v[1][-20:], b.table[1:], b.lens_dev[1:], torch.tensor([0, 20], dtype=torch.int32, device="cuda"))
    assert got is None and p.device_status() == 0
    held(b.run(p), ref, tol)


def test_refusals():
    p = pkg()
    b = Batch([40, 30], [2, 1], 8, 2, 64, 16)
    ok = dict(q=b.q, k_pages=b.k_pages, v_pages=b.v_pages, table=b.table, lens=b.lens_dev, scale=0.1, starts=b.starts)
    p.dispatch.attention_paged(**ok)
    bad = [dict(q=b.q.cpu()), dict(table=b.table.cpu()), dict(q=b.q.float()), dict(q=b.q[:, :, :32]), dict(q=b.q[0]), dict(q=b.q[:, :7]),
           dict(k_pages=b.k_pages[:, :, :8], v_pages=b.v_pages[:, :, :8]), dict(v_pages=b.v_pages[:1]), dict(lens=b.lens_dev.long()), dict(lens=b.lens_dev[:1]),
           dict(starts=b.starts[:2]), dict(table=b.table.long()), dict(starts=None), dict(max_new=0), dict(out=b.q.float()), dict(out=b.q[:1]),
           dict(k_pages=b.k_pages.transpose(1, 2), v_pages=b.v_pages.transpose(1, 2)), dict(q=b.q.half(), k_pages=b.k_pages.half(), v_pages=b.v_pages.half()),
           dict(q=b.q.repeat(1, 9, 1)), dict(out=b.q)]
    for change in bad:
        with pytest.raises(p.Ab2Error):
            p.dispatch.attention_paged(**{**ok, **change})
    assert p.dispatch.attention_paged(**{**ok, "q": b.q[:0], "starts": torch.zeros(3, dtype=torch.int32, device="cuda")}).shape == (0, 8, 64)


@pytest.mark.parametrize("new", [1, 4, 90])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_recorded_behind_copies_and_other_streams(new, dtype):
    """A call that is recorded behind a copy, a clear and another stream's work reads what they left: its launch may be set up before they have ended."""
    b = Batch([300, 95, 7], [new] * 3, 8, 2, 64, 16, dtype, seed=11, scatter=0.5)
    want = b.run(pkg())
    q = torch.zeros_like(b.q)
    run = lambda: pkg().dispatch.attention_paged(q, b.k_pages, b.v_pages, b.table, b.lens_dev, b.scale, b.starts)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        side.wait_stream(torch.cuda.current_stream())
        q.zero_()
        with torch.cuda.stream(side):
            half = torch.empty_like(b.q).copy_(b.q)
            for _ in range(20):
                half.mul_(2).mul_(0.5)   # exact, and slower than what the main stream does
        torch.cuda.current_stream().wait_stream(side)
        q.copy_(half)
        first, second = run(), run()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, want) and torch.equal(second, want)
    for _ in range(20):   # eager: behind kernels that have not ended
        q.zero_()
        q.copy_(b.q.mul(2)).mul_(0.5)
        got = run()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 20])
def test_a_long_f32_row_rounds_once_a_tile(new, dim):
    """Equal scores and equal values, all keys by one CTA (there is no workspace to cut the row by): the mean is the value itself, and every rounding of a
    sum goes the same way.  The weights are 1 and their sum is exact.  Values are summed over 32 keys, and those sums over n / 32 tiles: at most
    n / 32 + 32 roundings of 2^-24 each, and 4 more for the reciprocal, the product and the tile's last part.  One chain over the 20000 keys would be off by
    1.8e-4 (0.7 added to itself in f32), where 3.9e-5 is allowed."""
    n = 20000
    b = Batch([n], [new], 4, 2, dim, 256, F32, seed=1)
    b.q.zero_()
    b.v_pages.copy_(torch.where(torch.isnan(b.v_pages), b.v_pages, torch.full_like(b.v_pages, 0.7)))
    out = torch.empty_like(b.q)
    p = pkg()
    c, keep = p.dispatch._paged(b.k_pages, b.v_pages, b.table, b.lens_dev, b.starts, b.T)
    p.check(p.lib.ab2_paged_attention(C.byref(c), b.q.data_ptr(), 4 * dim, 4, out.data_ptr(), 4 * dim, new, b.scale, None, 0, p.dispatch.dtype_code(F32), torch.cuda.current_stream().cuda_stream))
    value = b.v_pages[~torch.isnan(b.v_pages)][0].double()
    assert ((out.double() / value - 1).abs() <= (n / 32 + 32 + 4) * 2.0 ** -24).all()


TALL = [(520, 8, 1, 128, 16), (300, 12, 4, 64, 64), (531, 5, 5, 128, 128), (180, 32, 2, 64, 32), (171, 30, 10, 128, 32), (90, 32, 1, 64, 256)]


@pytest.mark.parametrize("new,heads,kv_heads,dim,page", TALL)
def test_long_f32_chunks(new, heads, kv_heads, dim, page):
    """Rows of the tallest tiles: groups of 1 to 32 heads, with rows of no tokens, of no keys before them, and of a tile's last few tokens."""
    check(Batch([new, 0, new + 333, new + 1, 40], [new, 0, new, 1, 33], heads, kv_heads, dim, page, F32, seed=new))


@pytest.mark.parametrize("new,heads,kv_heads,dim,page", TALL)
def test_long_f32_chunks_out_of_sight(new, heads, kv_heads, dim, page):
    """Whatever the last 45 tokens hold, those before them answer the same bits."""
    b = Batch([new + 70], [new], heads, kv_heads, dim, page, F32, seed=7)
    want = b.run(pkg()).clone()
    seen = new - 45
    for bad_k, bad_v in ((math.nan, math.nan), (1.0, math.inf), (math.inf, 1.0), (torch.finfo(F32).min, -math.inf)):
        for pos in range(new + 70 - 45, new + 70):
            at = b.table[0, pos // page].item()
            b.k_pages[at, :, pos % page] = bad_k
            b.v_pages[at, :, pos % page] = bad_v
        got = b.run(pkg())
        assert torch.equal(got[:seen], want[:seen])
    assert pkg().device_status() == 0
