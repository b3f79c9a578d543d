"""How many bits a softmax weight and a query keep in attention over pages of 8 bits and through windows, as the header says it, kernel by kernel."""
import pytest
import torch

from helpers import pkg
from paged8_fixtures import LongBatch
from paged_fixtures import STEP, held

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def strict(b):
    """`LongBatch.expected` with a weight's own rounding in place of 2^-8: over codes f16's, 2^-11; over bf16 two bf16 terms, 2^-16, where a row's new tokens times the query heads of
    a KV head are at most 16, else 2^-8.  What f16 loses below its normal numbers: weights are kept at 8 times the unit or more where scales are of one size, and 2^-25 is 2^-28 of
    that, for each key.  Queries in e4m3 terms (2^-17.8 of their row's largest element) are counted only where the chunk kernel may answer the row: calls of more than 16 query rows.
    The sums of the tolerance are taken apart by the terms that a type or pages without scales do not have."""
    scales, sizes = b.scales, {}
    for dtype in (BF, F32):
        for plain in (False, True):
            b.dtype, b.scales = dtype, None if plain else scales
            ref, tol = b.expected()
            sizes[dtype, plain] = tol - ref.abs() * 1.01 * STEP[dtype]
    b.dtype, b.scales = BF, scales
    spread = (sizes[BF, True] - sizes[F32, True]) / 2.0 ** -8                         # sum p |v|
    lost = (sizes[BF, False] - sizes[F32, False] - 2.0 ** -8 * spread).clamp(min=0)    # by queries in terms
    group = b.heads // b.kv_heads
    if scales is not None:
        weight = torch.full((ref.shape[0], 1, 1), 2.0 ** -11 + max(b.lens) * 2.0 ** -28, dtype=torch.float64, device=ref.device)
    else:
        weight = torch.tensor([2.0 ** (-16 if m * group <= 16 else -8) for m in b.new for _ in range(m)], dtype=torch.float64, device=ref.device)[:, None, None]
    chunks = sum(b.new) * group > 16 if b.starts is not None else group > 16
    return ref, sizes[F32, False] + weight * spread + lost * chunks + ref.abs() * 1.01 * STEP[BF]


def check(b, **kw):
    ref, tol = strict(b)
    held(b.run(pkg(), **kw)[:ref.shape[0]], ref, tol)
    assert pkg().device_status() == 0


FORMS = [(True, 0, 0), (True, 150, 4), (False, 150, 4)]


@pytest.mark.parametrize("codes,window,sinks", FORMS)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(32, 8, 128, 16), (6, 2, 64, 32), (4, 4, 128, 64), (16, 1, 64, 16)])
def test_single_tokens(codes, window, sinks, heads, kv_heads, dim, page):
    lens = [1, 17, 64, 333, 700, 1290, 5000]
    check(LongBatch(lens, [1] * len(lens), heads, kv_heads, dim, page, BF, codes, window, sinks, one_each=True, scatter=0.7, seed=dim))


@pytest.mark.parametrize("codes,window,sinks", FORMS)
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(32, 8, 128, 16), (6, 2, 64, 32), (4, 4, 128, 64), (32, 1, 128, 128)])
@pytest.mark.parametrize("new,lens", [([9, 8, 17, 1], [9, 8, 150, 1]), ([40, 1, 0, 33], [333, 1290, 77, 33]), ([130, 257], [1130, 500]), ([4, 1], [2000, 5000]), ([2, 40, 1, 16, 4, 3], [90, 40, 2000, 300, 4, 1234])])
def test_chunks_and_short_rows(codes, window, sinks, heads, kv_heads, dim, page, new, lens):
    check(LongBatch(lens, new, heads, kv_heads, dim, page, BF, codes, window, sinks, scatter=0.7, seed=len(lens)))


@pytest.mark.parametrize("codes,window,sinks", FORMS)
@pytest.mark.parametrize("rows", [2, 40])   # one launch for all, and one of single tokens beside one of chunks
def test_a_single_token_alone_and_beside_a_chunk(codes, window, sinks, rows):
    """Within the formula's tolerance either way."""
    p = pkg()
    b = LongBatch([1500, 300] + [200 + r for r in range(rows - 2)], [1, 90] + [1] * (rows - 2), 8, 2, 128, 16, BF, codes, window, sinks, scatter=0.5, seed=3)
    ref, tol = strict(b)
    got = b.run(p)
    held(got, ref, tol)
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    alone = p.dispatch.attention_paged(b.q[:1].contiguous(), b.k_pages, b.v_pages, b.table[:1], b.lens_dev[:1], b.scale, one, scales=b.scales, window=window, sinks=sinks)
    held(alone, ref[:1], tol[:1])
