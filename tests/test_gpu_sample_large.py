"""Draws from vocabularies beyond 2^17 tokens, where a weight's unit is a larger part of the largest, and from rows that do not fit shared memory, against the definition in 64 bits."""
import math

import numpy as np
import pytest
import torch

from helpers import pkg

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def unit(vocab):
    """F, weights being whole numbers of 2^-F of the largest: 44, or what keeps the sum of a row's below 2^61."""
    return min(44, 61 - math.ceil(math.log2(vocab)))


def assert_drawn(got, z, u, T=1.0, k=0, p=1.0, least=0.0):
    """Each weight is off by 2^-30 of itself and half of a unit, so that a cumulative mass is by `off`, and f64 sums by less than the first again; top-p's border, by as much, moves the
    mass that stays by twice that.  The number times the mass lies between the token's bounds to that."""
    z = z.double().cpu().numpy()
    n = len(z)
    finite = z > -np.inf
    top = z[finite].max()
    w = np.where(finite, np.exp(np.where(finite, z - top, 0.0) / T), 0.0)
    order = np.lexsort((np.arange(n), -z))[:int(finite.sum())]
    if k > 0:
        order = order[:k]
    ws = w[order]
    up = np.cumsum(ws)
    off = n * 2.0 ** -(unit(n) + 1) + w.sum() * 2.0 ** -29
    right = False
    for nudge in (-off, off):
        m = len(order) if p >= 1 else max(1, min(len(order), int(np.searchsorted(up, p * up[-1] + nudge)) + 1))
        kept = np.zeros(n, dtype=bool)
        kept[order[:m]] = True
        kept &= w >= least * (1 - 2.0 ** -29)
        c = np.cumsum(np.where(kept, w, 0.0))
        right |= bool(kept[got]) and c[got] - w[got] - 4 * off <= u * c[-1] <= c[got] + 4 * off
    assert right, (got, u, T, k, p, least, off)


def draw(z, u, T=None, k=None, p=None, least=None):
    def dev(v, dtype=F32):
        return None if v is None else torch.full((z.shape[0],), v, dtype=dtype, device="cuda")
    got = pkg().dispatch.sample(z, torch.tensor(u, dtype=torch.float64).cuda(), dev(T), dev(k, torch.int32), dev(p), dev(least)).tolist()
    assert pkg().device_status() == 0
    return got


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("vocab,above", [(1 << 17, 24), ((1 << 17) + 1, 20), (1 << 20, 20), (1 << 24, 15), (1 << 24, 12)])
def test_a_tail_that_holds_much_of_the_mass(dtype, vocab, above):
    """One token above all others, which are alike (their weights' roundings all go one way) or differ a little."""
    g = torch.Generator(device="cuda").manual_seed(vocab)
    z = torch.stack([torch.full((vocab,), -0.3, device="cuda"), 0.5 * torch.randn(vocab, generator=g, device="cuda")]).to(dtype)
    z[:, vocab // 3] = above
    share = 1 / (1 + vocab * math.exp(-above))   # of the one, more or less
    us = [0.3 * (1 - share) / 3, 0.99 * (1 - share) / 3, 1 - 0.4 * (1 - share), 1 - 1e-5 * (1 - share)]
    for u in us:
        for row, got in enumerate(draw(z, [u, u])):
            assert_drawn(got, z[row], u)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("vocab", [600001, 1 << 20])
@pytest.mark.parametrize("first", [0, 1])   # on 16 bytes, and not
def test_rows_beyond_shared_memory(dtype, vocab, first):
    g = torch.Generator(device="cuda").manual_seed(vocab + first)
    z = (3 * torch.randn(3, vocab + 8, generator=g, device="cuda")).to(dtype)[:, first:first + vocab]
    z[1, ::3] = -math.inf
    z[2, :vocab // 2] = torch.finfo(dtype).min
    for i, rules in enumerate((dict(), dict(k=50), dict(k=5000), dict(k=300000, p=0.8), dict(p=0.9), dict(p=0.9, T=0.4), dict(p=0.999, least=0.001), dict(least=0.05), dict(T=1.7, k=700, p=0.5, least=0.02), dict(k=vocab))):
        u = [0.11 + 0.08 * i, 0.93 - 0.07 * i, (0.37 * i) % 1]
        for row, got in enumerate(draw(z, u, **rules)):
            f = {n: float(np.float32(v)) if n != "k" else v for n, v in rules.items()}
            assert_drawn(got, z[row], u[row], **f)


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("vocab", [600001])
def test_equal_logits_beyond_shared_memory(dtype, vocab):
    """Weights are exact: what stays are the first tokens."""
    z = torch.full((4, vocab), 1.5, dtype=dtype, device="cuda")
    u = [0.0, 0.25, 0.7, 0.999]
    for k, p in ((0, 1.0), (1, 1.0), (vocab // 2, 1.0), (0, 0.5), (vocab // 2, 0.25)):
        n = math.ceil(p * (k or vocab))
        assert draw(z, u, k=k, p=p) == [min(int(x * n), n - 1) for x in u]
