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
