"""The native module answers plain calls over pages of 8 bits, through windows and of the sampler as the Python side does, and leaves all others to it."""
import pytest
import torch

from helpers import pkg
from paged8_fixtures import LongBatch

pytestmark = pytest.mark.gpu


def both(monkeypatch, call):
    d = pkg().dispatch
    if d._fast is None:
        pytest.skip("the module was not built")
    one = call(d)
    with monkeypatch.context() as m:
        m.setattr(d, "_fast", None)
        two = call(d)
    return one, two


def test_same_answers(monkeypatch):
    for codes, window, sinks in ((True, 0, 0), (True, 50, 4), (False, 50, 0)):
        b = LongBatch([300, 40], [3, 1], 8, 2, 64, 16, torch.bfloat16, codes, window, sinks)
        call = lambda d: d.attention_paged(b.q, b.k_pages, b.v_pages, b.table, b.lens_dev, b.scale, b.starts, 3, scales=b.scales, window=window, sinks=sinks)  # noqa: E731
        one, two = both(monkeypatch, call)
        assert torch.equal(one, two)
        assert pkg().dispatch._fast.attention(b.q, b.k_pages, b.v_pages, b.table, b.lens_dev, b.scale, b.starts, 3, b.scales, window, sinks) is not None
    b = LongBatch([300, 40], [3, 1], 8, 2, 64, 16, torch.bfloat16, True)
    k, v = (torch.randn(4, 2, 64, device="cuda").bfloat16() for _ in range(2))
    f = pkg().dispatch.rotary_frequencies(64)
    kept = [t.clone() for t in (b.k_pages, b.v_pages, *b.scales)]

    def append(d):
        for t, was in zip((b.k_pages, b.v_pages, *b.scales), kept):
            t.view(torch.uint8).copy_(was.view(torch.uint8))
        q = d.paged_append(b.k_pages, b.v_pages, k, v, b.table, b.lens_dev, b.starts, b.q, f, scales=b.scales)
        return [q] + [t.view(torch.uint8).clone() for t in (b.k_pages, b.v_pages, *b.scales)]
    one, two = both(monkeypatch, append)
    assert all(torch.equal(x, y) for x, y in zip(one, two))
    z, u = torch.randn(5, 1000, device="cuda"), torch.rand(5, device="cuda")
    p = torch.full((5,), 0.7, device="cuda")
    one, two = both(monkeypatch, lambda d: d.sample(z, u, top_p=p))
    assert torch.equal(one, two) and pkg().dispatch._fast.sample(z, u, None, None, p, None) is not None


def test_what_is_not_plain_is_left_and_refused():
    p = pkg()
    d = p.dispatch
    if d._fast is None:
        pytest.skip("the module was not built")
    b = LongBatch([300, 40], [1, 1], 8, 2, 64, 16, torch.bfloat16, True, one_each=True)
    ks, vs = b.scales
    for scales, window, sinks in ((None, 0, 0), ((ks,), 0, 0), ((ks, vs[:-1]), 0, 0), ((ks, vs.double()), 0, 0), ((ks, vs.cpu()), 0, 0), ((ks, 3), 0, 0), ((ks, vs), -1, 0), ((ks, vs), 0, 4), ((ks, vs), 5, -1)):
        with pytest.raises((p.Ab2Error, AttributeError, TypeError)):
            d.attention_paged(b.q, b.k_pages, b.v_pages, b.table, b.lens_dev, b.scale, scales=scales, window=window, sinks=sinks)
    with pytest.raises(p.Ab2Error):
        d.attention_paged(b.q, b.k_pages.float().bfloat16(), b.v_pages.float().bfloat16(), b.table, b.lens_dev, b.scale, scales=b.scales)
    z, u = torch.randn(5, 1000, device="cuda"), torch.rand(5, device="cuda")
    assert d._fast.sample(z.t().contiguous().t(), u, None, None, None, None) is None
    for bad in (dict(uniforms=u.half()), dict(uniforms=u[:4]), dict(top_k=torch.ones(5, device="cuda")), dict(top_p=torch.ones(4, device="cuda")), dict(logits=z[0]), dict(logits=z.cpu())):
        args = dict(logits=z, uniforms=u)
        args.update(bad)
        with pytest.raises(p.Ab2Error):
            d.sample(**args)
