"""Attention over pages of 8 bits whose scales a caller made, down to the smallest that f32 has, in blocks behind larger and smaller ones."""
import pytest
import torch

from helpers import pkg
from paged8_fixtures import BLOCK, LongBatch
from paged_fixtures import held

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


def with_scales(b, exponents):
    """The batch with 2^exponents[i % len] for the scale of values of every row's block i."""
    scales = b.scales[1].clone()
    for r, n in enumerate(b.lens):
        b.v[r] = b.v[r].double()
        for j in range(0, n, BLOCK):
            page, at = b.table[r, j // b.page].item(), j % b.page // BLOCK
            to = 2.0 ** exponents[j // BLOCK % len(exponents)]
            b.v[r][j:j + BLOCK] *= to / scales[page, :, at].double()[None, :, None]
            scales[page, :, at] = to
    b.scales = (b.scales[0], scales)
    return b


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [[1, 1, 1], [2, 1, 2], [90, 1, 20]])
@pytest.mark.parametrize("exponents", [(-60, -119), (-66, -125), (-70, -120, -66, -118), (-119, -60), (-60, -119, -140), (-90, -91, -92, -117)])
def test_scales_below_those_that_the_append_makes(dtype, new, exponents):
    """Values are of the order of the largest scale: the tolerance counts half a step of bf16 (2^-8) of sum p |v|, and a block of 2^-57 of that or less may be there or not."""
    for heads, kv_heads, dim in ((8, 2, 128), (6, 2, 64)):
        b = with_scales(LongBatch([32, 90, 333], new if heads == 8 else [1, 1, 1], heads, kv_heads, dim, 32, dtype, scatter=0.5, seed=len(exponents)), exponents)
        ref, tol = b.expected()
        assert (tol < ref.abs().amax()).all()   # it tells a sum from twice that
        held(b.run(pkg()), ref, tol)
        assert pkg().device_status() == 0
