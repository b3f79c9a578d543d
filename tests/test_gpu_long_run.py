"""Decoding from a long context with its operators in a row - rotation and append to pages of 8 bits, attention through a window with first tokens, logits under rules, a token
drawn by given numbers - eagerly and as a recorded step, against the same in 64 bits; and calls at the ends of what is allowed."""
import math

import pytest
import torch

from helpers import pkg
from paged8_fixtures import LongBatch
from paged_fixtures import held, turned
from test_gpu_paged_run import D, H, KV, PAGE, VOCAB, Toy
from test_gpu_sample import allowed

pytestmark = pytest.mark.gpu
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("window,sinks", [(24, 3), (0, 0)])
def test_generation(recorded, window, sinks):
    """Keys and values are within an e4m3 step of those that came; what attention makes of them, and the token drawn, are those of the values that the cache holds.  f32 queries: the
    logits are off by some 1e-5, so that a token may differ from the one of the exact logits where u falls within 1e-4 of a border; those draws are few."""
    p = pkg()
    toy, rules = Toy(F32), (1.2, 0.1, 0.05)
    cache = p.PagedKVCache(40, PAGE, KV, D, batch=3, dtype="e4m3")
    prompts, rows, steps = [[5, 9, 2] * 25, [7], [1, 2, 3, 4] * 12], [2, 0, 1], 40
    device_rules = torch.tensor([rules] * 3, device="cuda")
    temperature, top_p, min_p = (torch.tensor(x, device="cuda") for x in ([0.7, 1.5, 1.0], [0.9, 1.0, 0.6], [0.0, 0.05, 0.01]))
    top_k = torch.tensor([0, 50, 20], dtype=torch.int32, device="cuda")
    uniforms, numbers = torch.zeros(3, device="cuda"), torch.rand(steps, 3, generator=torch.Generator().manual_seed(5))
    history = torch.full((3, 200), -1, dtype=torch.int32, device="cuda")
    for i, x in enumerate(prompts):
        history[i, :len(x)] = torch.tensor(x, dtype=torch.int32)
    lengths = torch.tensor([len(x) for x in prompts], dtype=torch.int32, device="cuda")

    def forward(step, ids):
        q, k, v = toy.parts(ids)
        q = cache.append(step, k, v, q=q, frequencies=toy.f)
        return cache.attention(step, q, 1 / math.sqrt(D), window=window, sinks=sinks)

    def choose(o):
        z = p.dispatch.adjust_logits(o.reshape(3, -1) @ toy.head.T, history, lengths, device_rules)
        return p.dispatch.sample(z, uniforms, temperature, top_k, top_p, min_p)

    def exact(row, ids):
        """Logits behind a sequence in f64, of the keys and values that the cache holds."""
        pos = torch.arange(len(ids), device="cuda")
        q, k, v = toy.parts(torch.tensor(ids, device="cuda"))
        q, k, v = turned(q, pos, toy.f)[-1], turned(k, pos, toy.f), v.double()
        kc, vc = (x.double() for x in cache.read(row))
        for came, got in ((k, kc), (v, vc)):   # codes of a block that grew: half a step, and half of the smallest step of a scale that is not above twice its largest / 224
            most = torch.stack([x.abs().amax((0, 2)) for x in came.split(16)]).repeat_interleave(16, 0)[:len(ids), :, None]
            assert ((got - came).abs() <= came.abs() * 2.0 ** -4 * 1.01 + most / 224 * 2.0 ** -10 * 2).all()
        kc, vc = (x.repeat_interleave(H // KV, dim=1) for x in (kc, vc))
        s = torch.einsum("hd,jhd->hj", q, kc) / math.sqrt(D)
        if window:
            s = s.masked_fill((len(ids) - 1 - pos >= window) & (pos >= sinks), -math.inf)
        z = toy.head.double() @ torch.einsum("hj,jhd->hd", torch.softmax(s, -1), vc).reshape(-1)
        count = torch.bincount(torch.tensor(ids, device="cuda"), minlength=VOCAB)
        return torch.where(count > 0, torch.where(z > 0, z / rules[0], z * rules[0]) - rules[1] - rules[2] * count, z)

    step = cache.step(rows, [len(x) for x in prompts], room=steps)
    o = forward(step, torch.tensor(sum(prompts, []), device="cuda"))
    cache.commit(step)
    uniforms.copy_(numbers[0])
    ids = choose(o[step.starts[1:].long() - 1]).long()
    seqs, other = [list(x) for x in prompts], 0

    def note(i):
        nonlocal other
        for r, t in enumerate(ids.tolist()):
            z, u = exact(rows[r], seqs[r]), numbers[i, r].double().item()
            args = (temperature[r].item(), top_k[r].item(), top_p[r].item(), min_p[r].item())
            if t not in allowed(z, u, *args):
                other += 1
                assert t in allowed(z, min(u + 1e-4, 1 - 1e-9), *args) | allowed(z, max(u - 1e-4, 0.0), *args) | allowed(z, u, args[0], args[1], args[2] + 1e-4, args[3]) | allowed(z, u, args[0], args[1], args[2] - 1e-4, args[3])
            seqs[r].append(t)
        history[torch.arange(3, device="cuda"), lengths.long()] = ids.int()
        lengths.add_(1)

    note(0)
    one = cache.step(rows, [1] * 3, room=steps)
    if recorded:
        static, chosen, graph, stream = ids.clone(), torch.empty(3, dtype=torch.int32, device="cuda"), torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=stream):   # recording runs nothing
            chosen.copy_(choose(forward(one, static)))
    for i in range(1, steps - 1):
        if i > 1:
            cache.step(rows, [1] * 3, into=one)
        uniforms.copy_(numbers[i])
        if recorded:
            static.copy_(ids)
            graph.replay()
            ids = chosen.long()
        else:
            ids = choose(forward(one, ids)).long()
        cache.commit(one)
        note(i)
    assert p.device_status() == 0 and [cache.seq_len(r) for r in rows] == [len(s) - 1 for s in seqs]
    assert other <= 3 and len(set(sum((s[-30:] for s in seqs), []))) > 10   # tokens are drawn, not one repeated


@pytest.mark.parametrize("codes", [True, False])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("window,sinks", [(16, 0), (31, 40), (200, 3)])
def test_rows_with_more_new_tokens_than_tokens(dtype, codes, window, sinks):
    for heads, kv_heads in ((8, 2), (4, 4), (1, 1)):
        b = LongBatch([10, 0, 355, 129, 1], [300, 7, 700, 140, 30], heads, kv_heads, 64, 16, dtype, codes, window, sinks, hide=False)
        ref, tol = b.expected()
        held(b.run(pkg()), ref, tol)
        assert pkg().device_status() == 0


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 1, 2], [90, 1, 130]])
@pytest.mark.parametrize("e", [-90, 90])
def test_queries_of_any_size(dtype, new, e):
    """Queries times 2^e under a scale of 2^-e are the same scores."""
    b = LongBatch([400, 90, 150], new, 8, 2, 128, 32, dtype, seed=6)
    b.q, b.scale = b.q * 2.0 ** e, b.scale * 2.0 ** -e
    b.q[1, 3] = 0
    ref, tol = b.expected()
    held(b.run(pkg()), ref, tol)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("new", [[1, 1], [90, 130]])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_a_query_that_is_not_finite_spoils_its_own_row_only(dtype, new, bad):
    b = LongBatch([400, 150], new, 8, 2, 128, 32, dtype, seed=8)
    ref, tol = b.expected()
    b.q[1, 3, 5] = bad
    got = b.run(pkg())
    assert got[1, 3].isnan().all()
    ref[1, 3], got[1, 3], tol[1, 3] = 0, 0, 0
    held(got, ref, tol)


def test_two_recorded_calls_have_workspaces_of_their_own():
    """Two captured calls that cut their rows, replayed on two streams at once, answer what each answers alone."""
    batches = [LongBatch([20000 + 700 * i, 9, 5000], [1, 1, 1], 8, 2, 128, 64, BF, True, 0, 0, seed=i, one_each=True) for i in range(2)]
    want, graphs, streams = [b.run(pkg()).clone() for b in batches], [], [torch.cuda.Stream() for _ in range(2)]
    for b, s in zip(batches, streams):
        out, g = torch.zeros_like(b.q), torch.cuda.CUDAGraph()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.graph(g, stream=s):
            b.run(pkg(), out=out)
        graphs.append((g, out))
    torch.cuda.synchronize()
    for _ in range(20):
        for (g, out), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (g, out), w in zip(graphs, want):
        assert torch.equal(out, w)
    assert pkg().device_status() == 0


def test_pages_behind_four_gigabytes():
    """Pages whose codes lie 2^32 bytes and more behind the pool's beginning, for the append and for every kernel of attention."""
    p, page, kv, dim = pkg(), 256, 8, 128
    pages = (2 ** 32 + 2 ** 29) // (page * kv * dim)
    pools, scales = [[torch.empty((pages, kv, page, dim), dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)], [torch.empty((pages, kv, page // 16), device="cuda") for _ in range(2)]]
    for dtype, new, window in ((BF, [1, 1], 0), (BF, [90, 1], 0), (BF, [90, 1], 300), (F32, [1, 40], 0)):
        b = LongBatch([700, 400], new, 32, kv, dim, page, dtype, True, window, 4 if window else 0, hide=False)
        ref, tol = b.expected()
        for big, small in zip(pools, (b.k_pages, b.v_pages)):
            big.view(torch.uint8)[-small.shape[0]:] = small.view(torch.uint8)
        for big, small in zip(scales, b.scales):
            big[-small.shape[0]:] = small
        shift = pages - b.k_pages.shape[0]
        b.table += shift
        b.k_pages, b.v_pages = pools
        b.scales = tuple(scales)
        held(b.run(p), ref, tol)
        assert p.device_status() == 0
        k = torch.randn(sum(new), kv, dim, device="cuda").to(dtype)
        low = [torch.zeros(b.k_pages.shape[0] - shift, kv, page, dim, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn) for _ in range(2)]
        low_scales = [torch.zeros(low[0].shape[0], kv, page // 16, device="cuda") for _ in range(2)]
        for big in pools:
            big.view(torch.uint8)[shift:] = 0
        for big in scales:
            big[shift:] = 0
        p.dispatch.paged_append(*low, k, 2 * k, b.table - shift, b.lens_dev, b.starts, scales=tuple(low_scales))
        p.dispatch.paged_append(*pools, k, 2 * k, b.table, b.lens_dev, b.starts, scales=tuple(scales))
        assert p.device_status() == 0
        for big, small in zip(pools, low):
            assert torch.equal(big.view(torch.uint8)[shift:], small.view(torch.uint8))
        for big, small in zip(scales, low_scales):
            assert torch.equal(big[shift:], small)


@pytest.mark.parametrize("codes,window", [(True, 0), (True, 90), (False, 90)])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("scale", [-0.11, 0.0])
def test_scales_of_scores_that_are_not_positive(dtype, codes, window, scale):
    for new in ([1, 1, 1], [90, 3, 260]):
        b = LongBatch([400, 90, 700], new, 8, 2, 128, 32, dtype, codes, window, 5 if window else 0, seed=9)
        b.scale = scale
        ref, tol = b.expected()
        held(b.run(pkg()), ref, tol)


def test_many_rows_draw():
    """More rows than CTAs at once, a cluster of one CTA each."""
    z = (2 * torch.randn(3000, 1200, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")).to(BF)
    u = torch.rand(3000, generator=torch.Generator().manual_seed(4))
    p = torch.full((3000,), 0.7, device="cuda")
    got = pkg().dispatch.sample(z, u.cuda(), top_p=p).tolist()
    for i in range(0, 3000, 37):
        assert got[i] in allowed(z[i], u[i].double().item(), p=p[i].double().item())
