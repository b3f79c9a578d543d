"""The native module leaves to dispatch.py what it does not take, with no error of its own behind."""
import pytest
import torch

from helpers import pkg


@pytest.mark.parametrize("layout", ["full", "", "\ud800", "half\0", None, 3])
def test_a_layout_that_is_none(layout):
    d = pkg().dispatch
    if d._fast is None:
        pytest.skip("the native module is not built")
    q, pos, f = torch.zeros(2, 2, 64), torch.zeros(2, dtype=torch.int32), torch.zeros(4, dtype=torch.float64)
    assert d._fast.rotary(q, None, pos, f, layout, 1.0) is None
    pages, table = torch.zeros(3, 2, 16, 64), torch.zeros(2, 2, dtype=torch.int32)
    assert d._fast.append(pages, pages, q, q, table, table[:, 0], None, None, None, layout, 1.0) is None
    with pytest.raises(pkg().Ab2Error):
        d.rotary_apply(q, None, pos, f, layout)
