"""Pages of 8 bits with scales that are no tensors are refused like all else, without a GPU."""
import pytest
import torch

from helpers import pkg


@pytest.mark.parametrize("other", [None, 3, 1.0, "scales", [1.0, 2.0]])
@pytest.mark.parametrize("codes", [True, False])
def test_scales_are_tensors(other, codes):
    p, z = pkg(), torch.zeros
    q, table, lens = z(2, 2, 64), z(2, 2, dtype=torch.int32), z(2, dtype=torch.int32)
    pages, s = z(3, 2, 32, 64).to(torch.float8_e4m3fn if codes else torch.float32), z(3, 2, 2)
    for scales in ((s, other), (other, s), [other, other]):
        for call in (lambda: p.dispatch.paged_append(pages, pages, q, q, table, lens, scales=scales), lambda: p.dispatch.attention_paged(q, pages, pages, table, lens, 1.0, scales=scales)):
            with pytest.raises(p.Ab2Error) as e:
                call()
            assert e.value.status == -7
