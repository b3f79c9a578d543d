"""Results of a serving step's operators that would share memory with what is still to be read are refused, to the byte: parts of one buffer that
lie between each other are served.  Refusals need no GPU; the calls that are served are tried on one."""
import ctypes as C
import random

import pytest
import torch

from helpers import pkg

BASE = 1 << 30
REFUSED = -7


def rotary(q, k, qo, ko, stride, out_stride, tokens=4, heads=4, kv=2, dim=64):
    """Byte offsets of f32 tensors, strides in elements."""
    return pkg().lib.ab2_rotary_apply(BASE + q, stride, heads, BASE + k, stride, kv, dim, 1 << 28, 0, tokens, 1 << 29, dim, 0, 1.0, BASE + qo, out_stride, BASE + ko, out_stride, 0, None)


def test_rotary_refuses_results_over_other_rows():
    S = 1000   # elements from a token to the next
    far = 1 << 24
    for q, k, qo, ko, out_stride in ((0, far, 4, 2 * far, S), (0, far, 4 * S, 2 * far, S), (0, far, 0, 2 * far, S + 1), (0, far, far, 2 * far, S), (0, far, 2 * far, 0, S), (0, far, 2 * far, 2 * far, S),
                                     (0, far, 2 * far, 2 * far + 1020, S), (0, far, 4 * (S - 255), 2 * far, S), (0, far, -4, 2 * far, S), (0, far, -4 * 3 * S, 2 * far, S), (0, far, 2 * far, far + 4 * S, 1024)):
        assert rotary(q, k, qo, ko, S, out_stride) == REFUSED, (q, k, qo, ko, out_stride)


def test_attention_append_and_logits_refuse():
    p = pkg()
    lib = p.lib
    c = p._lib.Paged(BASE, BASE + (1 << 20), 1 << 22, 1 << 23, 1 << 24, 4, 16, 2, 64, 3, 2, 5, 3)   # pools of 16 KB
    q = 1 << 26

    def attention(out, qs=512, os=512):
        return lib.ab2_paged_attention(C.byref(c), q, qs, 8, out, os, 3, 1.0, None, 0, 2, None)

    for out in (q, q + 16, q + 4 * 1024, q - 4 * 1024, q - 1024, BASE, BASE + 16, BASE + (1 << 20) + 16 * 1024 - 16):
        assert attention(out) == REFUSED, out
    assert attention(q + 1024, qs=1024, os=512) == REFUSED   # rows of other steps meet

    def append(qo, k=1 << 25, v=(1 << 25) + 4096, cache=c):
        return lib.ab2_paged_append(C.byref(cache), k, 128, v, 128, q, 512, 8, qo, 512, None, 0, 0, 1.0, 2, None)

    for qo in (q + 16, q - 1024, 1 << 25, (1 << 25) + 4096 + 1024, BASE + 4096, BASE + (1 << 20)):
        assert append(qo) == REFUSED, qo
    for v_pages in (BASE, BASE + 16 * 1024 - 16):
        same = p._lib.Paged(BASE, v_pages, 1 << 22, 1 << 23, 1 << 24, 4, 16, 2, 64, 3, 2, 5, 3)
        assert append(q, cache=same) == REFUSED

    def logits(out, stride=100):
        return lib.ab2_adjust_logits(BASE, stride, 3, 100, None, 0, 0, None, None, None, None, 0, None, BASE + out, 0, None)

    for out, stride in ((4, 100), (-4, 100), (400, 100), (0, 101), (0, 200), (400, 200)):
        assert logits(out, stride) == REFUSED, (out, stride)


def test_to_the_byte():
    """Rotary's refusal against every byte of every row."""
    rng = random.Random(4)
    refused = 0
    for _ in range(3000):
        tokens, es = rng.randint(1, 5), 4
        row = 2 * es   # one head of two elements
        steps = [rng.randint(2, 9) for _ in range(2)]
        if rng.random() < 0.5:
            steps[1] = steps[0]
        at = [0, rng.randint(-50, 50) * es]
        q, qo = ({BASE + at[i] + t * steps[i] * es + b for t in range(tokens) for b in range(row)} for i in range(2))
        in_place = at[0] == at[1] and (steps[0] == steps[1] or tokens == 1)
        want = bool(q & qo) and not in_place
        if not want and torch.cuda.is_available():
            continue   # it would be launched, on addresses that are nobody's
        rc = pkg().lib.ab2_rotary_apply(BASE + at[0], steps[0], 1, None, 0, 0, 2, 1 << 28, 0, tokens, 1 << 29, 2, 0, 1.0, BASE + at[1], steps[1], None, 0, 0, None)
        assert (rc == REFUSED) == want, (at, steps, tokens)
        refused += want
    assert refused > 300


@pytest.mark.gpu
def test_parts_of_one_buffer_are_served():
    p = pkg()
    d, T, H, KV, D = p.dispatch, 5, 4, 2, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    f, pos = d.rotary_frequencies(D), torch.arange(T, device="cuda")
    wide = torch.randn(T, H + 2 * KV + H, D, generator=g, device="cuda")
    q, k, spare = wide[:, :H], wide[:, H:H + KV], wide[:, H + 2 * KV:]
    want = d.rotary_apply(q.contiguous(), k.contiguous(), pos, f)
    d.rotary_apply(q, None, pos, f, out=(spare, None))   # a part of the same rows that no input is
    assert torch.equal(spare, want[0])
    d.rotary_apply(q, k, pos, f, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    with pytest.raises(p.Ab2Error):
        d.rotary_apply(q, k, pos, f, out=(wide[:, 1:1 + H], k))
    cache = p.PagedKVCache(4, 16, KV, D, dtype="f32")
    step = cache.step([0], [T])
    v = torch.randn(T, KV, D, generator=g, device="cuda")
    assert cache.append(step, k, v, q=q, out=q).data_ptr() == q.data_ptr()
    out = cache.attention(step, q, 0.1)
    assert torch.equal(cache.attention(step, q, 0.1, out=spare), out)
    with pytest.raises(p.Ab2Error):
        cache.attention(step, q, 0.1, out=wide[:, 2:2 + H])
    with pytest.raises(p.Ab2Error):
        cache.attention(step, q, 0.1, out=q)
    rows = torch.randn(4, 2, 300, generator=g, device="cuda")
    z = rows[:, 0]   # rows apart
    assert torch.equal(d.adjust_logits(z), z.contiguous())
    with pytest.raises(p.Ab2Error):
        d.adjust_logits(z, out=rows.view(-1)[:1200].view(4, 300))
    flat = z.contiguous()
    assert d.adjust_logits(flat, out=flat) is flat and p.device_status() == 0
