"""Plain calls of the serving step's operators go through the native module, others through dispatch.py's own look: the same kernels, the
same bits, the same refusals."""
import pytest
import torch

from helpers import pkg
from paged_fixtures import Batch

pytestmark = pytest.mark.gpu


def both(monkeypatch, call):
    d = pkg().dispatch
    assert d._fast is not None, "the native module is not built"
    one = call()
    with monkeypatch.context() as m:
        m.setattr(d, "_fast", None)
        two = call()
    return one, two


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("new", [1, 9])
def test_the_same_bits(monkeypatch, dtype, new):
    d = pkg().dispatch
    b = Batch([300, 20 + new], [new, new], 8, 2, 64, 16, dtype, seed=2, fill=0.0)
    f, pos = d.rotary_frequencies(64), torch.arange(b.T, device="cuda")
    k, v = torch.randn(b.T, 2, 64, device="cuda").to(dtype), torch.randn(b.T, 2, 64, device="cuda").to(dtype)
    assert d._fast.rotary(b.q, k, pos, f, "half", 1.0) is not None and d._fast.attention(b.q, b.k_pages, b.v_pages, b.table, b.lens_dev, 0.1, b.starts, None) is not None
    for one, two in (both(monkeypatch, lambda: d.rotary_apply(b.q, k, pos, f, "interleaved", 1.1)), both(monkeypatch, lambda: d.rotary_apply(b.q, None, pos.int(), f)),
                     both(monkeypatch, lambda: (b.run(pkg()), b.run(pkg(), max_new=new)))):
        for x, y in zip(one, two):
            assert x is y is None or torch.equal(x, y)

    def append(**kw):
        out = d.paged_append(b.k_pages, b.v_pages, k, v, b.table, b.lens_dev, b.starts, **kw)
        return out, b.k_pages.clone(), b.v_pages.clone()
    for kw in (dict(), dict(q=b.q, frequencies=f, magnitude=2), dict(frequencies=f, layout="interleaved")):
        for x, y in zip(*both(monkeypatch, lambda: append(**kw))):
            assert x is y is None or torch.equal(x, y)
    z, h, r = torch.randn(2, 999, device="cuda").to(dtype), torch.randint(0, 999, (2, 30), device="cuda", dtype=torch.int32), torch.rand(2, 3, device="cuda") + 0.5
    ids, val, n = torch.randint(0, 999, (2, 3), device="cuda", dtype=torch.int32), torch.randn(2, 3, device="cuda"), torch.tensor([30, 4], dtype=torch.int32, device="cuda")
    allowed = d.allowed_words(torch.rand(2, 999, device="cuda") < 0.5)
    assert d._fast.logits(z, h, n, r, ids, val, allowed) is not None
    for args in ((z,), (z, h, None, r), (z, h, n, r, ids, val), (z, None, None, None, ids, val, allowed), (z, h, n, r, ids, val, allowed)):
        one, two = both(monkeypatch, lambda: d.adjust_logits(*args))
        assert torch.equal(one, two)
    assert pkg().device_status() == 0


def test_what_is_not_plain_is_left_to_the_other(monkeypatch):
    d = pkg().dispatch
    f, pos = d.rotary_frequencies(64), torch.arange(4, device="cuda")
    q = torch.randn(4, 8, 64, device="cuda")
    for bad in (q.cpu(), q[:, :4], q.double(), q[0], "q", None):
        assert d._fast.rotary(bad, None, pos, f, "half", 1.0) is None
    for args in ((q, q[:2], pos, f, "half", 1.0), (q, None, pos[:3], f, "half", 1.0), (q, None, pos.float(), f, "half", 1.0), (q, None, pos, f.float(), "half", 1.0), (q, None, pos, f, "full", 1.0),
                 (q, None, pos, f, "half", "1"), (q, None, pos, f, None, 1.0), (q, None, pos, d.rotary_frequencies(66), "half", 1.0), (q,), ()):
        assert d._fast.rotary(*args) is None
    out = d.rotary_apply(torch.nn.Parameter(q), None, pos, f)[0]
    assert torch.equal(out, d.rotary_apply(q, None, pos, f)[0]) and not out.requires_grad
    # refused by the library itself: the same status from both
    b = Batch([40], [2], 8, 2, 64, 16, fill=0.0)
    wide = b.q.repeat(1, 9, 1)
    statuses = []
    for fast in (d._fast, None):
        monkeypatch.setattr(d, "_fast", fast)
        with pytest.raises(pkg().Ab2Error) as e:
            d.attention_paged(wide, b.k_pages, b.v_pages, b.table, b.lens_dev, 0.1, b.starts, 2)
        statuses.append((e.value.status, str(e.value)))
    assert statuses[0] == statuses[1] and statuses[0][0] == -1
