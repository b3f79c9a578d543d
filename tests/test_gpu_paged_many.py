"""Attention over a paged cache of batches that mix many rows: prompts of a tile or less, single tokens, rows without tokens, chunks."""
import pytest
import torch

from helpers import pkg
from paged_fixtures import Batch, held

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("heads,kv_heads,dim", [(32, 8, 128), (8, 8, 128), (16, 1, 64), (32, 1, 128)])
@pytest.mark.parametrize("rows,longest", [(30, 64), (30, 130), (32, 17), (300, 90)])
def test_many_short_prompts(rows, longest, heads, kv_heads, dim):
    """A CTA has several pieces of one tile of keys, or of one for its first tile of rows and two for its second."""
    lens = [1 + (longest - 1) * (1 + 13 * r % 17) // 17 for r in range(rows)]
    b = Batch(lens, lens, heads, kv_heads, dim, 16, BF, seed=rows)
    ref, tol = b.expected()
    first = b.run(pkg())
    held(first, ref, tol)
    for _ in range(20):
        assert torch.equal(b.run(pkg()), first)
    assert pkg().device_status() == 0


def mixed(rows, heads, kv_heads, dim, page, dtype=BF, ctx=300, chunk=70):
    """Rows with no new token, 1, 4, 5 and chunks, in turns, behind contexts of all lengths up to `ctx`; the last row is a chunk."""
    new = [[1, 0, 4, 1, 5, chunk, 1, 17][r % 8] for r in range(rows - 1)] + [chunk + 3]
    lens = [n + ctx * (r * 7 % 23) // 22 if n else (r * 5 % 3) * 10 for r, n in enumerate(new)]
    return Batch(lens, new, heads, kv_heads, dim, page, dtype, seed=rows, extra=2)


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 16), (16, 1, 64, 32), (6, 2, 64, 16), (20, 1, 128, 64)])
@pytest.mark.parametrize("rows", [31, 32, 33, 34, 64, 65, 128, 129, 425])
def test_single_tokens_and_chunks_of_many_rows(rows, heads, kv_heads, dim, page):
    """One launch serves all up to a number of rows (128, 64 and 32 of the first three kinds of heads); of more, the few-token rows and the chunks have a launch each, which
    leave out the other's."""
    p, b = pkg(), mixed(rows, heads, kv_heads, dim, page)
    n = b.starts_list[-1]
    ref, tol = b.expected()
    for bound in (None, max(b.new), 1, 4):
        out = torch.full_like(b.q, 7.0)
        held(b.run(p, max_new=bound, out=out)[:n], ref, tol)
        assert (out[n:] == 7).all() and p.device_status() == 0
    first = b.run(p)[:n]
    for _ in range(10):
        assert torch.equal(b.run(p)[:n], first)


@pytest.mark.parametrize("rows,ctx", [(33, 3000), (40, 6000)])
def test_both_launches_cut_their_rows(rows, ctx):
    """One workspace for both: the second launch's pieces lie where the first one's lay."""
    b = mixed(rows, 32, 8, 128, 64, ctx=ctx, chunk=150)
    ref, tol = b.expected()
    for _ in range(3):
        held(b.run(pkg())[:b.starts_list[-1]], ref, tol)
    assert pkg().device_status() == 0


@pytest.mark.parametrize("rows", [32, 33, 400])
def test_recorded_with_many_rows(rows):
    """Recorded once, replayed with other lengths and other new tokens: rows change from one launch's to the other's."""
    p = pkg()
    a = mixed(rows, 8, 2, 128, 16)
    b = mixed(rows, 8, 2, 128, 16)
    swapped = list(reversed(b.new))
    b = Batch([n + (r * 11 % 200) for r, n in enumerate(swapped)], swapped, 8, 2, 128, 16, seed=5, extra=2)
    pages, width = max(x.k_pages.shape[0] for x in (a, b)), max(x.table.shape[1] for x in (a, b))
    k, v = (torch.zeros((pages, 2, 16, 128), dtype=BF, device="cuda") for _ in range(2))
    table, lens, starts = torch.zeros((rows, width), dtype=torch.int32, device="cuda"), torch.zeros_like(a.lens_dev), torch.zeros_like(a.starts)
    q, out, graph = torch.zeros_like(a.q), torch.zeros_like(a.q), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p.dispatch.attention_paged(q, k, v, table, lens, a.scale, starts, max(a.new), out)
    for x in (a, b, a):
        k[:x.k_pages.shape[0]], v[:x.v_pages.shape[0]], table[:, :x.table.shape[1]] = x.k_pages, x.v_pages, x.table
        lens.copy_(x.lens_dev), starts.copy_(x.starts), q.copy_(x.q)
        graph.replay()
        torch.cuda.synchronize()
        held(out[:x.starts_list[-1]], *x.expected())
    assert p.device_status() == 0


@pytest.mark.parametrize("rows", [33, 400])
def test_f32_of_many_rows(rows):
    b = mixed(rows, 6, 2, 64, 16, F32)
    held(b.run(pkg())[:b.starts_list[-1]], *b.expected())
    assert pkg().device_status() == 0
