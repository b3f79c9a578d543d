"""A decoder of one attention layer served from a paged cache, its operators in a row: rotation and append, attention, logits under
rules, the greedy choice - eagerly and as a recorded step - against the same in 64 bits; and sessions with rules."""
import math

import numpy as np
import pytest
import torch

from helpers import pkg
from model_fixtures import SMALL, build_pair
from paged_fixtures import turned

pytestmark = pytest.mark.gpu
H, KV, D, VOCAB, PAGE = 8, 2, 64, 500, 16


class Toy:
    """Token -> q, k, v rows of a table; attention; a head over its output."""

    def __init__(self, dtype):
        g = torch.Generator(device="cuda").manual_seed(11)
        self.embed = torch.randn(VOCAB, (H + 2 * KV) * D, generator=g, device="cuda").to(dtype)
        self.head = (torch.randn(VOCAB, H * D, generator=g, device="cuda") / 8).to(dtype)
        self.f = pkg().dispatch.rotary_frequencies(D, 10000.0, pkg().dispatch.RotaryScaling("linear", 2.0))

    def parts(self, ids):
        x = self.embed[ids]
        return x[:, :H * D].view(-1, H, D), x[:, H * D:(H + KV) * D].view(-1, KV, D), x[:, (H + KV) * D:].view(-1, KV, D)

    def exact(self, ids, counted, rules):
        """Logits after a whole sequence, in f64."""
        q, k, v = self.parts(torch.tensor(ids, device="cuda"))
        pos = torch.arange(len(ids), device="cuda")
        q, k, v = turned(q, pos, self.f)[-1], turned(k, pos, self.f), v.double()
        k, v = (x.repeat_interleave(H // KV, dim=1) for x in (k, v))
        p = torch.softmax(torch.einsum("hd,jhd->hj", q, k) / math.sqrt(D), -1)
        z = self.head.double() @ torch.einsum("hj,jhd->hd", p, v).reshape(-1)
        count = torch.bincount(torch.tensor(counted, device="cuda"), minlength=VOCAB)
        return torch.where(count > 0, torch.where(z > 0, z / rules[0], z * rules[0]) - rules[1] - rules[2] * count, z)


@pytest.mark.parametrize("recorded", [False, True])
def test_generation_over_a_paged_cache(recorded):
    p, dtype = pkg(), torch.float32
    toy, rules = Toy(dtype), (1.3, 0.2, 0.1)
    cache = p.PagedKVCache(30, PAGE, KV, D, batch=3, dtype="f32")
    prompts = [[5, 9, 2] * 11, [7], [1, 2, 3, 4] * 5]
    rows, steps = [2, 0, 1], 40
    device_rules = torch.tensor([rules] * 3, device="cuda")
    history = torch.full((3, 200), -1, dtype=torch.int32, device="cuda")
    for i, x in enumerate(prompts):
        history[i, :len(x)] = torch.tensor(x, dtype=torch.int32)
    lengths = torch.tensor([len(x) for x in prompts], dtype=torch.int32, device="cuda")

    def forward(step, ids):
        q, k, v = toy.parts(ids)
        q = cache.append(step, k, v, q=q, frequencies=toy.f)
        return cache.attention(step, q, 1 / math.sqrt(D))

    def choose(o):
        return p.dispatch.argmax(p.dispatch.adjust_logits(o.reshape(3, -1) @ toy.head.T, history, lengths, device_rules))

    step = cache.step(rows, [len(x) for x in prompts], room=steps)
    o = forward(step, torch.tensor(sum(prompts, []), device="cuda"))
    cache.commit(step)
    ends = step.starts[1:].long() - 1
    ids = choose(o[ends]).long()
    seqs, margins = [list(x) for x in prompts], []

    def note():
        for i, t in enumerate(ids.tolist()):
            z = toy.exact(seqs[i], seqs[i], rules)
            top = torch.topk(z, 2)
            margins.append((top.values[0] - top.values[1]).item())
            assert t == top.indices[0].item() or margins[-1] < 1e-3, f"token {t} instead of {top.indices[0].item()} by {margins[-1]}"
            seqs[i].append(t)
        history[torch.arange(3, device="cuda"), lengths.long()] = ids.int()
        lengths.add_(1)

    note()
    one = cache.step(rows, [1] * 3, room=steps)
    if recorded:
        static, chosen, graph, stream = ids.clone(), torch.empty(3, dtype=torch.int32, device="cuda"), torch.cuda.CUDAGraph(), torch.cuda.Stream()
        k0, v0 = cache.k.clone(), cache.v.clone()
        with torch.cuda.graph(graph, stream=stream):
            chosen.copy_(choose(forward(one, static)))
        cache.k.copy_(k0), cache.v.copy_(v0)
    for i in range(steps - 2):
        if i:
            cache.step(rows, [1] * 3, into=one)
        if recorded:
            static.copy_(ids)
            graph.replay()
            ids = chosen.long()
        else:
            ids = choose(forward(one, ids)).long()
        cache.commit(one)
        note()
    assert p.device_status() == 0 and [cache.seq_len(r) for r in rows] == [len(s) - 1 for s in seqs]
    k, _ = cache.read(rows[0])
    want = turned(toy.parts(torch.tensor(seqs[0][:-1], device="cuda"))[1], torch.arange(len(seqs[0]) - 1, device="cuda"), toy.f)
    assert (k - want).abs().max() < 1e-5
    assert sorted(margins)[len(margins) // 2] > 1e-2   # the choices are not ties
    cache.truncate(3, rows[0])
    cache.truncate(0, rows[1])
    assert cache.free_pages() == 30 - 1 - len(cache._pages[rows[2]])


def test_sessions_with_rules():
    """A session without rules answers as before; penalties, biases and a grammar change what it picks as the formula says."""
    p = pkg()
    model = build_pair(SMALL, "int8_channel", capacity=64)[0]
    R = p.sessions.LogitRules
    prompt = [3, 1, 4, 1, 5]

    def run(rules):
        engine = p.sessions.SessionEngine(model, max_batch=1, capacity=64)
        s = engine.prepare_session_with_chunk_size(prompt, 12, rules=rules)
        seen = []
        while not s.finished:
            seen.append(s.next_logits.double().cpu().numpy().copy())
            engine.advance(s)
            if not s.finished:
                engine.decode_sessions([s])
        return s.generated_ids, seen

    plain, _ = run(None)
    assert run(R())[0] == plain
    got, logits = run(R(repetition=1.7, presence=0.3, frequency=0.2))
    for i, (t, z) in enumerate(zip(got, logits)):
        count = np.bincount(prompt + got[:i], minlength=z.size)
        z = np.where(count > 0, np.where(z > 0, z / 1.7, z * 1.7) - 0.3 - 0.2 * count, z)
        assert z[t] >= z.max() - 1e-5
    assert run(R(bias={17: 1e4}))[0] == [17] * 12
    only = run(R(allowed=lambda ids: [2 + len(ids), 30]))[0]
    assert all(t in (2 + i, 30) for i, t in enumerate(only))
    with pytest.raises(p.Ab2Error):
        R(repetition=0.0)
    with pytest.raises(p.Ab2Error):
        run(R(allowed=lambda ids: [10 ** 6]))
    for nothing in ([], [False] * SMALL["vocab"]):
        with pytest.raises(p.Ab2Error):
            run(R(allowed=lambda ids: nothing))
    assert run(R(allowed=lambda ids: None))[0] == plain
