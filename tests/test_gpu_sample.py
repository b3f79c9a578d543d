"""Sampling from given random numbers against its definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

from helpers import pkg

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def allowed(z, u, T=1.0, k=0, p=1.0, least=0.0):
    """The tokens that may be the answer for one row: one, but where u or p falls on a border between two by less than what weights are off.  A weight is a table's power of two
    (rounded to 31 bits: 2^-32) times e^v as a whole number of 2^-31 (2^-32, and its float 2^-33), their product cut to 31 bits (2^-31): 2^-30.4 of it together, less than 2^-30; then
    it is rounded to a whole number of 2^-44 of the largest, half of one for each token.  f64 sums of up to 2^20 terms: 2^-33."""
    z = z.double().cpu().numpy()
    valid = np.nonzero(z > -np.inf)[0]
    if len(valid) == 0:
        return {-1}
    top = z[valid].max()
    with np.errstate(all="ignore"):
        x = np.where(z[valid] == top, 0.0, (top - z[valid]) / T) if T > 0 else np.where(z[valid] == top, 0.0, np.inf)
    w = np.exp(-x)
    order = np.lexsort((valid, -z[valid]))
    if not T > 0 or least > 1:
        k = 1
    if 0 < k < len(order):
        order = order[:k]
    off = len(z) * 2.0 ** -44 + w.sum() * 2.0 ** -30
    answers = set()
    ws = w[order]
    up = np.cumsum(ws)
    for nudge in (-off, off):
        m = len(order)
        if p < 1:
            m = int(np.searchsorted(up, max(p, 0.0) * up[-1] + nudge)) + 1
        m = max(1, min(m, len(order)))
        kept = np.sort(valid[order[:m]][(ws[:m] >= min(least, 1.0)) | (np.arange(m) == 0)])
        c = np.cumsum(w[np.searchsorted(valid, kept)])
        for more in (-off, 0.0, off):
            answers.add(int(kept[min(max(int(np.searchsorted(c, u * c[-1] + more, side="right")), 0), len(kept) - 1)]))
    return answers


def check(z, u, T=None, k=None, p=None, least=None):
    def dev(v, dtype):
        return None if v is None else torch.tensor(v, dtype=dtype).cuda()
    rows = z.shape[0]
    got = pkg().dispatch.sample(z, torch.as_tensor(u).cuda(), dev(T, F32), dev(k, torch.int32), dev(p, F32), dev(least, F32)).tolist()
    us = torch.as_tensor(u).double().tolist()
    narrow = 0
    f = lambda v, i, d: d if v is None else float(np.float32(v[i]))  # noqa: E731
    for i in range(rows):
        may = allowed(z[i], us[i], f(T, i, 1.0), 0 if k is None else k[i], f(p, i, 1.0), f(least, i, 0.0))
        narrow += len(may) > 1
        assert got[i] in may, (i, got[i], may, us[i], f(T, i, 1.0), None if k is None else k[i], f(p, i, 1.0), f(least, i, 0.0))
    assert narrow <= max(2, rows // 50)   # the tolerance decides next to nothing
    assert pkg().device_status() == 0
    return got


def rules(rng, rows, vocab):
    T = [float(rng.choice([0.3, 0.7, 1.0, 1.3, 3.0])) for _ in range(rows)]
    k = [int(rng.choice([0, 0, 1, 2, 40, 300, vocab, 2 * vocab])) for _ in range(rows)]
    p = [float(rng.choice([1.0, 1.0, 0.95, 0.9, 0.5, 0.1, 0.999])) for _ in range(rows)]
    least = [float(rng.choice([0.0, 0.0, 0.02, 0.1, 0.5])) for _ in range(rows)]
    return T, k, p, least


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("vocab", [1, 2, 7, 33, 500, 2047, 4097, 8192, 32000, 50257, 128256])
@pytest.mark.parametrize("rows", [1, 6, 40])
def test_rules_of_all_kinds(dtype, vocab, rows):
    g = torch.Generator(device="cuda").manual_seed(vocab + rows)
    rng = np.random.default_rng(vocab + rows)
    z = (torch.randn(rows, vocab, generator=g, device="cuda") * 3).to(dtype)
    check(z, torch.rand(rows, generator=g, device="cuda"), *rules(rng, rows, vocab))
    check(z, torch.rand(rows, generator=g, device="cuda", dtype=torch.float64))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_one_rule_at_a_time(dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    z = (torch.randn(24, 32000, generator=g, device="cuda") * 2).to(dtype)
    u = torch.rand(24, generator=g, device="cuda", dtype=torch.float64)
    for k in (1, 5, 1000, 5000, 31999):
        check(z, u, k=[k] * 24)
        check(z, u, k=[k] * 24, p=[0.9] * 24)
        check(z, u, k=[k] * 24, least=[0.01] * 24)
        check(z, u, k=[k] * 24, p=[0.7] * 24, least=[0.3] * 24)
    for p in (0.0, 1e-6, 0.3, 0.9, 0.9999, 1.0, 2.0, -1.0):
        check(z, u, p=[p] * 24)
        check(z, u, p=[p] * 24, least=[0.05] * 24)
    for least in (1e-7, 0.2, 1.0, 3.0):
        check(z, u, least=[least] * 24)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab", [500, 30000, 128256])
def test_equal_logits_go_by_index(dtype, vocab):
    """Weights are exact there: what stays is a prefix of the indices."""
    rows = 12
    u = torch.linspace(0, 0.999, rows, dtype=torch.float64)
    z = torch.full((rows, vocab), 1.5, dtype=dtype, device="cuda")
    k = [0, 1, 7, vocab // 2, vocab - 1, vocab] * 2
    p = [1.0] * 6 + [0.3] * 6
    got = pkg().dispatch.sample(z, u.cuda(), None, torch.tensor(k, dtype=torch.int32).cuda(), torch.tensor(p).cuda()).tolist()
    for i in range(rows):
        n = k[i] or vocab
        if p[i] < 1:
            n = math.ceil(float(np.float32(p[i])) * n)
        assert got[i] == min(int(u[i].item() * n), n - 1), (i, got[i], n)
    # a few high ones among many equal ones, and two values
    z[:, 5], z[:, vocab - 3] = 3.0, 2.0
    check(z, u, k=k, p=p)
    z = torch.where(torch.arange(vocab, device="cuda") % 3 == 0, 1.0, 0.5).to(dtype).expand(rows, vocab).contiguous()
    check(z, u, k=k, p=p)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
def test_masks_and_values_that_are_not_finite(dtype):
    g = torch.Generator(device="cuda").manual_seed(9)
    z = (torch.randn(9, 1000, generator=g, device="cuda") * 3).to(dtype)
    z[0] = -math.inf                       # nothing is left
    z[1] = math.nan
    z[2, 1:] = -math.inf                   # one is
    z[3, :999] = -math.inf
    z[4, ::2] = math.nan
    z[5, 7], z[5, 300] = math.inf, math.inf
    z[6] = torch.finfo(dtype).min          # the type's lowest value is a logit as any other
    z[7] = torch.where(torch.arange(1000, device="cuda") < 900, torch.finfo(dtype).min, z[7].float()).to(dtype)
    z[8, 100:900] = -math.inf
    for u in (0.0, 0.3, 0.999999):
        for kw in ({}, dict(k=[3] * 9), dict(p=[0.8] * 9), dict(least=[0.1] * 9), dict(T=[0.2] * 9, k=[20] * 9, p=[0.9] * 9)):
            got = check(z, [u] * 9, **kw)
            assert got[:4] == [-1, -1, 0, 999] and got[5] in (7, 300)


def test_temperatures_at_their_ends():
    g = torch.Generator(device="cuda").manual_seed(4)
    z = torch.randn(10, 5000, generator=g, device="cuda")
    z[:, 77] = z[:, 4000] = 9.0
    u = torch.rand(10, generator=g, device="cuda")
    for T in (0.0, -1.0, math.nan):
        assert pkg().dispatch.sample(z, u, torch.full((10,), T, device="cuda")).tolist() == [77] * 10
    for T in (1e-30, 1e-4, 50.0, 1e4, 1e30):
        got = check(z, u, T=[T] * 10, k=[0, 1, 5, 0, 0, 100, 0, 4999, 0, 0], p=[1.0, 1.0, 1.0, 0.5, 1.0, 0.9, 0.99, 1.0, 0.2, 1.0], least=[0.0] * 8 + [0.5, 0.9])
        assert T > 1 or set(got) <= {77, 4000}


def test_numbers_at_their_ends():
    z = torch.randn(8, 3000, device="cuda")
    u = [0.0, 1.0 - 2.0 ** -53, 1.0, 2.0, -1.0, math.nan, 2.0 ** -60, 0.5]
    for kw in ({}, dict(k=[10] * 8)):
        got = pkg().dispatch.sample(z, torch.tensor(u, dtype=torch.float64).cuda(), **{n: torch.tensor(v, dtype=torch.int32).cuda() for n, v in (("top_k", kw["k"]),)} if kw else {}).tolist()
        assert all(0 <= t < 3000 for t in got)
        for i in (0, 1, 6, 7):
            assert got[i] in allowed(z[i], u[i], k=10 if kw else 0)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rows_that_lie_apart(dtype):
    g = torch.Generator(device="cuda").manual_seed(2)
    for cols, first in ((777, 0), (1003, 1), (9000, 8)):
        wide = torch.randn(5, cols + 21, generator=g, device="cuda").to(dtype)
        z = wide[:, first:first + cols]
        u = torch.rand(5, generator=g, device="cuda")
        rng = np.random.default_rng(cols)
        check(z, u, *rules(rng, 5, cols))
        a, b = (pkg().dispatch.sample(x, u, top_p=torch.full((5,), 0.9, device="cuda")) for x in (z, z.contiguous()))
        assert torch.equal(a, b)


def test_rows_share_nothing_and_runs_are_the_same():
    """A row's token does not hang on how many rows there are, and so on how many CTAs have a row."""
    g = torch.Generator(device="cuda").manual_seed(8)
    z = torch.randn(300, 20000, generator=g, device="cuda") * 2
    u = torch.rand(300, generator=g, device="cuda")
    rng = np.random.default_rng(1)
    T, k, p, least = (torch.tensor(v, dtype=torch.int32 if j == 1 else F32).cuda() for j, v in enumerate(rules(rng, 300, 20000)))
    whole = pkg().dispatch.sample(z, u, T, k, p, least)
    for _ in range(3):
        assert torch.equal(whole, pkg().dispatch.sample(z, u, T, k, p, least))
    for n in (1, 3, 17, 33, 74):
        assert torch.equal(whole[:n], pkg().dispatch.sample(z[:n], u[:n], T[:n], k[:n], p[:n], least[:n]))


def test_large_vocabulary_and_what_comes_out():
    g = torch.Generator(device="cuda").manual_seed(8)
    for vocab in (300001, 1 << 20):
        z = torch.randn(2, vocab, generator=g, device="cuda")
        check(z, [0.2, 0.9], k=[0, 50], p=[0.9, 1.0])
        check(z, [0.2, 0.9], k=[0, 60000], p=[1.0, 0.8])


def test_frequencies_are_those_of_the_distribution():
    """Numbers on a grid of 4096: a token comes out as often as its probability says, to one either way for each border of a kept token."""
    z = torch.tensor([0.3, -1.0, 2.0, 1.9, -4.0, 0.0], device="cuda").repeat(4096, 1)
    u = (torch.arange(4096, dtype=torch.float64, device="cuda") + 0.5) / 4096
    got = torch.bincount(pkg().dispatch.sample(z, u, top_k=torch.full((4096,), 5, dtype=torch.int32, device="cuda")).long(), minlength=6).double()
    want = torch.softmax(z[0].double().masked_fill(torch.arange(6, device="cuda") == 4, -math.inf), 0) * 4096
    assert ((got - want).abs() <= 1.0).all()


def test_recorded_call_and_another_stream():
    g = torch.Generator(device="cuda").manual_seed(8)
    z, u, out = torch.randn(4, 9000, generator=g, device="cuda"), torch.zeros(4, device="cuda"), torch.zeros(4, dtype=torch.int32, device="cuda")
    p = torch.full((4,), 0.8, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        pkg().dispatch.sample(z, u, top_p=p, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            assert pkg().dispatch.sample(z, u, top_p=p, out=out) is out
        for x in (0.1, 0.6, 0.99):
            u.fill_(x)
            graph.replay()
            s.synchronize()
            for i in range(4):
                assert out[i].item() in allowed(z[i], u[i].double().item(), p=float(np.float32(0.8)))


def test_sessions_draw():
    from model_fixtures import SMALL, build_pair
    p = pkg()
    model = build_pair(SMALL, "int8_channel", capacity=64)[0]
    S = p.sessions.Sampling

    def run(*samplings):
        engine = p.sessions.SessionEngine(model, max_batch=len(samplings), capacity=64)
        live = [engine.prepare_session_with_chunk_size([3, 1, 4], 12, sampling=s) for s in samplings]
        while any(not s.finished for s in live):
            for s in live:
                engine.advance(s)
            engine.decode_sessions([s for s in live if not s.finished])
        return [s.generated_ids for s in live]
    greedy, cold, one, hot = run(None, S(temperature=0.0), S(temperature=5.0, top_k=1), S(temperature=3.0, seed=1))
    assert greedy == cold == one and hot != greedy
    assert run(S(temperature=3.0, seed=1))[0] == hot and run(S(temperature=3.0, seed=2))[0] != hot


@pytest.mark.parametrize("vocab", [700, 20000, 128256])
@pytest.mark.parametrize("least", [0.0, 0.03])
def test_top_p_over_logits_of_all_kinds(vocab, least):
    """Log-probabilities, logits next to zero and about it, far from it, few that differ: what top-p keeps ends on ties, near zero, or anywhere."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    n = lambda: torch.randn(vocab, generator=g, device="cuda")  # noqa: E731
    few = torch.zeros(vocab, device="cuda")
    few[:5] = torch.tensor([4.0, 3.0, 2.0, 1.0, -1.0])
    z = torch.stack([torch.log_softmax(3 * n(), 0), n() * 1e-6, n() * 1e-3, few + n() * 1e-30, few - 1e-5, (3 * n()).round(), 300 * n(), 1000 + n(), -1000 - n().abs(), -n().abs() * 1e-20, n() - 7.0, few * 20]).to(BF)
    rows = z.shape[0]
    for p, T in ((0.9, 1.0), (0.5, 0.7), (0.99, 3.0), (0.2, 1.0), (0.9999, 1.0)):
        check(z, torch.rand(rows, generator=torch.Generator().manual_seed(vocab + int(100 * p))).tolist(), [T] * rows, None, [p] * rows, [least] * rows)
