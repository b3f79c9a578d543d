"""Attention over a paged bf16 cache carries the weights of rows of up to 16 query rows a KV head in two bf16 terms, whichever kernel serves them, and counts
every key once."""
import pytest
import torch

from helpers import pkg
from paged_fixtures import STEP, Batch, held

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def strict(b):
    """`Batch.expected` with 2^-16 for a weight in place of 2^-8 where a row's new tokens times the query heads of a KV head are at most 16: rounded to bf16 a weight is off by 2^-8 of itself at most, and what that left, rounded again, by 2^-8
    of 2^-8.  The tolerances of both element types are sums of the same terms but for the weight's (2^-8 of sum p |v|) and the output's own."""
    ref, loose = b.expected()
    b.dtype = F32
    _, tight = b.expected()
    b.dtype = BF
    own = ref.abs() * 1.01
    spread = ((loose - own * STEP[BF]) - (tight - own * STEP[F32])) / 2.0 ** -8   # sum p |v|
    weight = torch.tensor([2.0 ** (-16 if m * (b.heads // b.kv_heads) <= 16 else -8) for m in b.new for _ in range(m)], dtype=torch.float64, device=ref.device)
    return ref, (tight - own * STEP[F32]) + weight[:, None, None] * spread + own * STEP[BF]


def check(b, **kw):
    ref, tol = strict(b)
    held(b.run(pkg(), **kw)[:ref.shape[0]], ref, tol)
    assert pkg().device_status() == 0


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(32, 8, 128, 16), (6, 2, 64, 32), (4, 4, 128, 64), (16, 1, 64, 16), (32, 1, 128, 128)])
@pytest.mark.parametrize("new,lens", [([1, 1, 1], [700, 64, 3]), ([9, 8, 17, 1], [9, 8, 150, 1]), ([40, 1, 0, 33], [333, 1290, 77, 33]), ([130, 257], [1130, 500]), ([4, 1], [2000, 5000]), ([2, 40, 1, 16, 4, 3], [90, 40, 2000, 300, 4, 1234])])
def test_weights_in_two_terms(heads, kv_heads, dim, page, new, lens):
    check(Batch(lens, new, heads, kv_heads, dim, page, seed=len(lens), scatter=0.7))


@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (20, 1)])
def test_a_single_token_does_not_depend_on_who_shares_its_batch(heads, kv_heads):
    """Alone, among single tokens, and beside a chunk: its answer is within the same tolerance, and within twice that of the others."""
    p, ctx = pkg(), 1500
    beside = Batch([ctx, 300], [1, 90], heads, kv_heads, 128, 16, seed=3, scatter=0.5)
    ref, tol = strict(beside)
    got = beside.run(p)
    held(got, ref, tol)
    one = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    alone = p.dispatch.attention_paged(beside.q[:1].contiguous(), beside.k_pages, beside.v_pages, beside.table[:1], beside.lens_dev[:1], beside.scale, one)
    held(alone, ref[:1], tol[:1])
    held(alone, got[:1].double(), 2 * tol[:1])


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,lens", [([1], [2300]), ([1] * 40, [700 + 9 * r for r in range(40)]), ([4, 1], [900, 1333]), ([200, 1], [1500, 2100]), ([513], [513]), ([1] * 39 + [130], [300 + 11 * r for r in range(40)])])
def test_every_key_counts_once(dtype, dim, new, lens):
    """Equal scores, and values that are 1 in one dimension for one key: a token's answer there is 1 / (keys it sees), or 0 if the key is not among them.  A key lost or
    doubled at the end of a page, a tile, a unit or a CTA's run answers 0 or twice as much.  Weights of equal scores are 1 and exact; the sum of the weights is a whole
    number below 2^24 and exact, its reciprocal and the product round to 2^-24 each, and pieces are joined with factors of 1; then half a step of the output."""
    p = pkg()
    b = Batch(lens, new, 4, 2, dim, 16, dtype, seed=dim, fill=0.0)
    b.q.zero_()
    pos = torch.cat([torch.arange(n - m, n, device="cuda") for n, m in zip(lens, new)])
    row = torch.cat([torch.full((m,), r, device="cuda") for r, m in enumerate(new)])
    d = torch.arange(dim, device="cuda")
    table = b.table.long()
    for start in range(0, max(lens), dim):
        b.v_pages.zero_()
        for r, n in enumerate(lens):
            j = torch.arange(start, max(start, min(n, start + dim)), device="cuda")
            b.v_pages[table[r, j // 16], :, j % 16, j - start] = 1
        got = b.run(p).double()
        want = torch.where(start + d[None, :] <= pos[:, None], 1.0 / (pos[:, None] + 1).double(), torch.zeros((), dtype=torch.float64, device="cuda"))[:, None]
        assert ((got - want).abs() <= want * (STEP[dtype] * 1.01 + 2.0 ** -22)).all(), (start, row[((got - want).abs() > want * 0.1).any(-1).any(-1)].unique().tolist())
    assert p.device_status() == 0
