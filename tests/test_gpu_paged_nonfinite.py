"""Inf and NaN among the values that a query sees, and among those that it does not, behind long contexts and with many queries."""
import math

import pytest
import torch

from helpers import pkg
from paged_fixtures import Batch, held

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def put(b, row, pos, dim, value):
    b.v_pages[b.table[row, pos // b.page].item(), :, pos % b.page, dim] = value
    b.v[row][pos, :, dim] = value


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64), (20, 1, 128)])
@pytest.mark.parametrize("new,ctx", [(1, 9000), (3, 2500), (90, 3000), (600, 1100), (300, 0)])
def test_a_value_reaches_those_that_see_it_in_its_dimension(dtype, heads, kv_heads, dim, new, ctx):
    """An Inf early in the context answers Inf in its dimension, a NaN NaN, whatever else is there; all other dimensions are what they were.  The last
    token's values are NaN in a dimension of their own, which the tokens before it do not see."""
    p = pkg()
    b = Batch([ctx + new, 40], [new, 1], heads, kv_heads, dim, 32, dtype, seed=new, scatter=0.5)
    put(b, 0, 0, 3, math.inf)
    put(b, 0, 0, 7, math.nan)
    put(b, 0, 0, 9, math.inf)
    put(b, 0, ctx // 2, 9, -math.inf)
    put(b, 0, ctx + new - 1, 11, math.nan)
    ref, tol = b.expected()
    got = b.run(p)
    assert (got[:new, :, 3] == math.inf).all() and torch.isnan(got[:new, :, 7]).all() and torch.isnan(got[new - 1, :, 11]).all()
    if ctx:
        assert torch.isnan(got[:new, :, 9]).all()
    else:   # both at the first position: the one that was put there last
        assert (got[:new, :, 9] == -math.inf).all()
    fine = [d for d in range(dim) if d not in (3, 7, 9, 11)]
    held(got[:, :, fine], ref[:, :, fine], tol[:, :, fine])
    held(got[:new - 1, :, 11], ref[:new - 1, :, 11], tol[:new - 1, :, 11])
    held(got[new:], ref[new:], tol[new:])
    assert p.device_status() == 0


@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (8, 8, 64)])
def test_rows_computed_again_beside_others(heads, kv_heads, dim):
    """Several chunks in one call, some with hidden NaN, some with visible Inf: each answers as alone, and every time the same bits."""
    p = pkg()
    new, lens = [130, 1, 200, 7, 64, 300], [900, 5000, 200, 700, 3000, 333]
    b = Batch(lens, new, heads, kv_heads, dim, 16, BF, seed=6, scatter=0.5)
    put(b, 0, 899, slice(None), math.nan)
    put(b, 2, 199, slice(0, 8), math.inf)
    put(b, 4, 100, 5, math.inf)
    ref, tol = b.expected()
    first = b.run(p)
    s = b.starts_list
    fine = torch.ones_like(first, dtype=torch.bool)
    fine[s[1] - 1] = False                   # the token that sees the NaN
    fine[s[3] - 1, :, :8] = False
    fine[s[4]:s[5], :, 5] = False
    assert torch.isnan(first[s[1] - 1]).all() and (first[s[4]:s[5], :, 5] == math.inf).all() and (first[s[3] - 1, :, :8] == math.inf).all()
    held(first[fine], ref[fine], tol[fine])
    for _ in range(5):
        assert torch.equal(b.run(p)[fine], first[fine])
    assert p.device_status() == 0
