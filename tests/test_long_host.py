"""Pages of 8 bits, windows and sampling without a GPU: what the entry points refuse, how a cache of 8 bits keeps its scales, and sessions that draw."""
import ctypes as C

import pytest
import torch

from helpers import pkg
from test_paged_host import cache
from test_sessions_host_logic import FakeModel

E4 = torch.float8_e4m3fn
GOOD = dict(k_pages=1 << 20, v_pages=1 << 21, table=1 << 22, lens=1 << 23, starts=1 << 24, pages=4, page_size=32, kv_heads=2, head_dim=64, table_width=3, rows=2, tokens=5, table_stride=3)
# at GOOD: a pool is 4 * 32 * 2 * 64 = 16384 codes, its scales 4 * 2 * 2 of 4 bytes


def paged(**kw):
    return pkg()._lib.Paged(**{**GOOD, **kw})


SHAPES = ((dict(k_pages=None), -7), (dict(v_pages=None), -7), (dict(table=None), -7), (dict(lens=None), -7), (dict(page_size=24), -8), (dict(page_size=8), -8), (dict(page_size=512), -8),
          (dict(head_dim=96), -8), (dict(pages=0), -1), (dict(rows=0), -1), (dict(tokens=-1), -1), (dict(table_width=0), -1), (dict(table_stride=2), -1), (dict(kv_heads=0), -1),
          (dict(starts=None), -1), (dict(k_pages=(1 << 20) + 8), -2))


def test_attention_refuses_before_any_device_work():
    lib = pkg().lib

    def window(c, window=9, sinks=2, q=1 << 25, qs=512, heads=8, out=1 << 26, os=512, max_new=3, dtype=2, work=None):
        return lib.ab2_paged_attention_window(C.byref(c) if c else None, window, sinks, q, qs, heads, out, os, max_new, 1.0, work, 0, dtype, None)

    def codes(c, ks=1 << 27, vs=1 << 28, window=0, sinks=0, q=1 << 25, qs=512, heads=8, out=1 << 26, os=512, max_new=3, dtype=2, work=None):
        return lib.ab2_paged_attention_e4m3(C.byref(c) if c else None, ks, vs, window, sinks, q, qs, heads, out, os, max_new, 1.0, work, 0, dtype, None)

    for call in (window, codes):
        assert call(None) == -7 and call(paged(tokens=0)) == 0
        for kw, code in SHAPES:
            assert call(paged(**kw)) == code, kw
        for kw, code in ((dict(window=-1), -1), (dict(window=0, sinks=1), -1), (dict(window=4, sinks=-1), -1), (dict(window=(1 << 30) + 1), -1), (dict(window=1, sinks=(1 << 30) + 1), -1), (dict(q=None), -7),
                         (dict(out=None), -7), (dict(heads=7), -1), (dict(heads=0), -1), (dict(heads=66), -1), (dict(out=1 << 25), -7), (dict(max_new=0), -1), (dict(qs=511), -1), (dict(os=100), -1),
                         (dict(qs=513), -2), (dict(q=(1 << 25) + 2), -2), (dict(dtype=1), -3), (dict(dtype=9), -3), (dict(work=(1 << 25) + 8), -2)):
            assert call(paged(), **kw) == code, kw
    for kw, code in ((dict(ks=None), -7), (dict(vs=None), -7), (dict(ks=None, vs=None), -7), (dict(ks=(1 << 27) + 2), -2), (dict(vs=(1 << 28) + 1), -2), (dict(out=1 << 27), -7), (dict(out=(1 << 28) + 48), -7),
                     (dict(out=(1 << 21) + 16368), -7)):
        assert codes(paged(), **kw) == code, kw


def test_append_refuses_before_any_device_work():
    lib = pkg().lib

    def append(c, ks=1 << 27, vs=1 << 28, k=1 << 25, kst=128, v=1 << 26, vst=128, q=None, qst=0, heads=0, qo=None, qos=0, f=None, rot=0, layout=0, dtype=2):
        return lib.ab2_paged_append_e4m3(C.byref(c) if c else None, ks, vs, k, kst, v, vst, q, qst, heads, qo, qos, f, rot, layout, 1.0, dtype, None)

    assert append(None) == -7 and append(paged(tokens=0)) == 0
    for kw, code in SHAPES:
        assert append(paged(**kw)) == code, kw
    q = dict(q=1 << 29, qst=256, heads=4, qo=1 << 30, qos=256)
    for kw, code in ((dict(ks=None), -7), (dict(vs=None), -7), (dict(ks=None, vs=None), -7), (dict(ks=(1 << 27) + 2), -2), (dict(vs=(1 << 28) + 3), -2), (dict(k=None), -7), (dict(v=None), -7),
                     (dict(kst=127), -1), (dict(vst=5), -1), (dict(k=(1 << 25) + 1), -2), (dict(dtype=1), -3), (dict(dtype=7), -3), (dict(layout=2), -7), (dict(rot=66, f=1 << 31), -1), (dict(rot=3, f=1 << 31), -1),
                     (dict(rot=8), -7), (dict(**q) | dict(qo=None), -7), (dict(**q) | dict(qst=255), -1), (dict(heads=-1), -1),
                     # pages, scales and the rest lie apart
                     (dict(vs=1 << 27), -7), (dict(vs=(1 << 27) + 60), -7), (dict(ks=(1 << 20) + 16380), -7), (dict(vs=1 << 21), -7), (dict(ks=1 << 25), -7), (dict(vs=(1 << 26) + 4), -7), (dict(k=1 << 20), -7),
                     (dict(v=(1 << 21) + 64), -7), (dict(**q) | dict(qo=1 << 27), -7), (dict(**q) | dict(q=1 << 28, qo=1 << 28), -7)):
        assert append(paged(), **kw) == code, kw


def test_sampling_refuses_before_any_device_work():
    lib = pkg().lib

    def sample(z=1 << 20, st=100, rows=2, vocab=100, u=1 << 21, wide=0, T=None, k=None, p=None, least=None, out=1 << 22, dtype=0):
        return lib.ab2_sample(z, st, rows, vocab, u, wide, T, k, p, least, out, dtype, None)

    assert sample(rows=0) == 0
    for kw, code in ((dict(z=None), -7), (dict(u=None), -7), (dict(out=None), -7), (dict(st=99), -1), (dict(vocab=0), -1), (dict(vocab=-4), -1), (dict(rows=-1), -1), (dict(vocab=(1 << 24) + 1, st=1 << 25), -8),
                     (dict(rows=1 << 28), -8), (dict(dtype=5), -3), (dict(z=(1 << 20) + 2), -2), (dict(u=(1 << 21) + 4, wide=1), -2), (dict(u=(1 << 21) + 2), -2), (dict(T=1), -2), (dict(k=2), -2), (dict(p=3), -2),
                     (dict(least=5), -2), (dict(out=(1 << 22) + 1), -2), (dict(out=(1 << 20) + 796), -7), (dict(out=1 << 21), -7), (dict(out=(1 << 21) + 12, wide=1), -7), (dict(T=1 << 22), -7), (dict(k=(1 << 22) + 4), -7),
                     (dict(p=(1 << 22) - 4), -7), (dict(least=1 << 22), -7)):
        assert sample(**kw) == code, kw


def test_cpu_tensors_and_wrong_scales_are_refused():
    p = pkg()
    d, z = p.dispatch, torch.zeros
    q, i32 = z(2, 2, 64), lambda *s: z(*s, dtype=torch.int32)  # noqa: E731
    pages, wide, s = z(3, 2, 32, 64).to(E4), z(3, 2, 32, 64), z(3, 2, 2)
    calls = [lambda: d.paged_append(pages, pages, q, q, i32(2, 2), i32(2), scales=(s, s)), lambda: d.attention_paged(q, pages, pages, i32(2, 2), i32(2), 1.0, scales=(s, s)),
             lambda: d.attention_paged(q, wide, wide, i32(2, 2), i32(2), 1.0, window=3, sinks=1), lambda: d.sample(z(2, 9), z(2)),
             lambda: d.sample(z(2, 9), z(2), z(2), i32(2), z(2), z(2), i32(2))]
    for call in calls:
        with pytest.raises(p.Ab2Error) as e:
            call()
        assert e.value.status == -7 and "CUDA device" in str(e.value)
    for scales, kv in ((None, pages), (s, pages), ((s,), pages), ((s, s, s), pages), ((s, s[:, :1]), pages), ((s, z(3, 2, 1)), pages), ((s.double(), s), pages), ((s, z(3, 2, 4)[:, :, ::2]), pages), ((s, s), wide),
                       ((s, s), pages[0])):
        with pytest.raises(p.Ab2Error):
            d.paged_append(kv, kv, q, q, i32(2, 2), i32(2), scales=scales)
        with pytest.raises(p.Ab2Error):
            d.attention_paged(q, kv, kv, i32(2, 2), i32(2), 1.0, scales=scales)


def test_a_cache_of_8_bits():
    c = cache(20, 32, 4, dtype="e4m3", n_layers=3)
    assert c.k.dtype == c.v.dtype == E4 and c.k.shape == (3, 20, 2, 32, 64)
    assert c.k_scales.shape == c.v_scales.shape == (3, 20, 2, 2) and c.k_scales.dtype == torch.float32
    assert cache().k_scales is None
    c.commit(c.step([1], [40]))
    g = torch.Generator().manual_seed(1)
    codes, scales = torch.randn(3, 20, 2, 32, 64, generator=g).to(E4), torch.exp2(torch.randint(-9, 9, (3, 20, 2, 2), generator=g).float())
    c.k.copy_(codes), c.k_scales.copy_(scales), c.v.copy_(codes), c.v_scales.copy_(2 * scales)
    k, v = c.read(1, layer=2)
    assert k.shape == v.shape == (40, 2, 64)
    for t in range(40):
        at = c._pages[1][t // 32]
        want = codes[2, at, :, t % 32].float() * scales[2, at, :, t % 32 // 16, None]
        assert torch.equal(k[t], want) and torch.equal(v[t], 2 * want)


def test_sessions_draw_by_their_own_rules(monkeypatch):
    """Each session's numbers come from its own seed, in order; one without a rule stays greedy."""
    mod = pkg().sessions
    asked = []

    def last_max(logits):
        v = logits.float()
        return (v.shape[-1] - 1 - torch.flip(v, [-1]).argmax(-1)).to(torch.int32)

    def drawn(logits, uniforms, temperature=None, top_k=None, top_p=None, min_p=None, out=None):
        one = lambda t: None if t is None else t.item()  # noqa: E731
        assert logits.shape[0] == 1 and uniforms.shape == (1,) and 0 <= uniforms.item() < 1
        asked.append((uniforms.item(), one(temperature), one(top_k), one(top_p), one(min_p)))
        return torch.tensor([7], dtype=torch.int32)

    monkeypatch.setattr(mod, "argmax", last_max)
    monkeypatch.setattr(mod, "sample", drawn)
    S = mod.Sampling

    def run(sampling):
        asked.clear()
        engine = mod.SessionEngine(FakeModel(), max_batch=1, capacity=64)
        s = engine.prepare_session_with_chunk_size([1, 2], 5, sampling=sampling)
        while not s.finished:
            engine.advance(s)
            if not s.finished:
                engine.decode_sessions([s])
        return s.generated_ids, list(asked)
    ids, calls = run(None)
    assert calls == [] and ids == [3, 4, 5, 6, 7]
    ids, calls = run(S(temperature=0.5, top_k=3, top_p=0.9, min_p=0.25, seed=4))
    assert ids == [7] * 5 and len({c[0] for c in calls}) == 5
    assert all(c[1] == 0.5 and c[2] == 3 and abs(c[3] - 0.9) < 1e-7 and c[4] == 0.25 for c in calls)
    assert run(S(temperature=0.5, top_k=3, top_p=0.9, min_p=0.25, seed=4))[1] == calls
    assert run(S(seed=5))[1][0][0] != calls[0][0]
