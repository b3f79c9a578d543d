"""Chunks over pages of 8 bits in which a block's values are far smaller than its neighbours': right, and not paid for by all rows that see it."""
import pytest
import torch

from helpers import pkg
from paged8_fixtures import LongBatch
from paged_fixtures import held
from test_gpu_paged_small_scales import with_scales

pytestmark = pytest.mark.gpu
BF = torch.bfloat16


@pytest.mark.parametrize("heads,kv_heads,dim,page", [(8, 2, 128, 32), (6, 2, 64, 16), (32, 1, 128, 64)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (100, 5)])
@pytest.mark.parametrize("exponents", [(-20, 0, 0, 0, 0, 0, 0), (0, -16), (0, -15, -30, 3), (-58, 0, 1, 2, -40, 20), (-80, -80, -80, -80, -80, 0)])
def test_blocks_far_apart(heads, kv_heads, dim, page, window, sinks, exponents):
    """Rows that see small blocks alone, large ones alone, and both: each is held to half a step of bf16 of sum p |v| of its own."""
    b = with_scales(LongBatch([700, 130, 90], [600, 130, 20], heads, kv_heads, dim, page, BF, True, window, sinks, scatter=0.5, seed=len(exponents), hide=False), exponents)
    ref, tol = b.expected()
    held(b.run(pkg()), ref, tol)
    assert pkg().device_status() == 0


def test_a_block_far_below_its_neighbours_costs_no_second_pass():
    """A row over again by itself takes some hundred times as long as by the tensor cores; rows of which the small block is next to nothing are a few per cent slower, and a factor of 4 is far from either."""
    times = []
    for exponents in ((0,) * 50, (0,) * 49 + (-20,)):
        b = with_scales(LongBatch([6000], [2000], 16, 4, 128, 64, BF), exponents)
        for _ in range(3):
            b.run(pkg())
        took = []
        for _ in range(9):
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            b.run(pkg())
            end.record()
            end.synchronize()
            took.append(start.elapsed_time(end))
        times.append(sorted(took)[4])
    assert times[1] < 4 * times[0], times
