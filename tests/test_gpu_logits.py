"""The rules of a sampler on logits against their formula in 64 bits."""
import math

import pytest
import torch

from helpers import pkg
from paged_fixtures import held, rounded_off

pytestmark = pytest.mark.gpu
BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def expected(logits, history=None, lengths=None, rules=None, ids=None, values=None, mask=None):
    """In f64, with how far f32 arithmetic and one rounding may be off: four operations, each 2^-24 of what it works on."""
    z, size = logits.double().cpu(), logits.double().cpu().abs()
    rows, vocab = z.shape
    for r in range(rows):
        if history is not None:
            h = history[r].cpu()[:int(lengths[r]) if lengths is not None else None]
            h = h[(h >= 0) & (h < vocab)].long()
            count = torch.bincount(h, minlength=vocab).double()
            rho, presence, frequency = rules[r].double().cpu()
            new = torch.where(z[r] > 0, z[r] / rho, z[r] * rho)
            off = presence + frequency * count
            size[r] = torch.where(count > 0, new.abs() + presence.abs() + frequency.abs() * count, size[r])
            z[r] = torch.where(count > 0, new - off, z[r])
        if ids is not None:
            last = {}
            for i, b in zip(ids[r].tolist(), values[r].double().tolist()):
                if 0 <= i < vocab:
                    last[i] = b
            for i, b in last.items():
                z[r, i] += b
                size[r, i] += abs(b)
        if mask is not None:
            z[r][~mask[r].cpu()] = -math.inf
    return z, 6 * 2.0 ** -24 * size + rounded_off(z.nan_to_num(posinf=0.0, neginf=0.0), logits.dtype)


def agree(got, ref, tol):
    got = got.double().cpu()
    fine = torch.isfinite(ref)
    assert torch.equal(got[~fine], ref[~fine])
    held(got[fine], ref[fine], tol[fine])


@pytest.mark.parametrize("dtype", [BF, F16, F32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 31), (2, 1000), (1, 32000), (5, 8192), (2, 128256), (3, 4099), (70, 600)])
@pytest.mark.parametrize("parts", ["history", "bias", "mask", "all", "none"])
def test_rules(dtype, rows, vocab, parts):
    p = pkg()
    g = torch.Generator(device="cuda").manual_seed(vocab)
    logits = (torch.randn(rows, vocab, generator=g, device="cuda") * 4).to(dtype)
    args = {}
    if parts in ("history", "all"):
        n = 700
        args["history"] = torch.randint(-3, vocab + 3, (rows, n), generator=g, device="cuda", dtype=torch.int32)
        args["history"][:, ::3] = torch.randint(0, min(vocab, 9), (rows, (n + 2) // 3), generator=g, device="cuda", dtype=torch.int32)
        args["lengths"] = torch.randint(0, n + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
        args["lengths"][0] = n
        args["rules"] = torch.rand(rows, 3, generator=g, device="cuda") + 0.5
        args["rules"][-1] = torch.tensor([1.0, 0.0, 0.0])
    ids = values = mask = None
    if parts in ("bias", "all"):
        ids = torch.randint(-2, vocab + 2, (rows, 33), generator=g, device="cuda", dtype=torch.int32)   # some twice, some outside
        values = torch.randn(rows, 33, generator=g, device="cuda")
    if parts in ("mask", "all"):
        mask = torch.rand(rows, vocab, generator=g, device="cuda") < 0.6
        mask[-1] = False   # nothing is left of a row
    got = p.dispatch.adjust_logits(logits, bias_ids=ids, bias_values=values, allowed=p.dispatch.allowed_words(mask) if mask is not None else None, **args)
    ref, tol = expected(logits, args.get("history"), args.get("lengths"), args.get("rules"), ids, values, mask)
    agree(got, ref, tol)
    again = logits.clone()   # in place
    assert p.dispatch.adjust_logits(again, bias_ids=ids, bias_values=values, allowed=p.dispatch.allowed_words(mask) if mask is not None else None, out=again, **args) is again
    assert torch.equal(again, got)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_infinities_nan_and_the_lowest_value(dtype):
    p = pkg()
    low = torch.finfo(dtype).min
    logits = torch.tensor([[math.inf, -math.inf, math.nan, low, -low, 0.0, -0.0, 1.0] * 8], device="cuda").to(dtype)
    mask = torch.ones(1, 64, dtype=torch.bool, device="cuda")
    mask[0, :16] = False
    got = p.dispatch.adjust_logits(logits, allowed=p.dispatch.allowed_words(mask))
    assert (got[0, :16] == -math.inf).all()   # whatever they held
    assert torch.equal(got[0, 16:].nan_to_num(nan=5.0, posinf=6.0, neginf=7.0), logits[0, 16:].nan_to_num(nan=5.0, posinf=6.0, neginf=7.0))
    history = torch.arange(64, dtype=torch.int32, device="cuda")[None]
    got = p.dispatch.adjust_logits(logits, history, None, torch.tensor([[2.0, 0.0, 0.0]], device="cuda"))
    first = got[0, :8].float().tolist()
    assert first[0] == math.inf and first[1] == -math.inf and math.isnan(first[2]) and first[3] == -math.inf
    assert first[4] == -low / 2 and first[5] == 0 and first[6] == 0 and first[7] == 0.5


def test_rows_apart_and_offsets_off_the_boundary():
    p = pkg()
    wide = torch.randn(4, 3, 1000, device="cuda")
    ids = torch.tensor([[3], [4], [5], [6]], dtype=torch.int32, device="cuda")
    values = torch.ones(4, 1, device="cuda")
    want = p.dispatch.adjust_logits(wide[:, -1].contiguous(), bias_ids=ids, bias_values=values)
    assert torch.equal(p.dispatch.adjust_logits(wide[:, -1], bias_ids=ids, bias_values=values), want)
    flat = torch.empty(4001, device="cuda")
    flat[1:] = wide[:, -1].reshape(-1)
    assert torch.equal(p.dispatch.adjust_logits(flat[1:].view(4, 1000), bias_ids=ids, bias_values=values), want)
    h = torch.zeros(4, 50, dtype=torch.int32, device="cuda")[:, ::2]
    r = torch.tensor([[1.5, 0.1, 0.2]] * 4, device="cuda")
    assert torch.equal(p.dispatch.adjust_logits(wide[:, 0], h, None, r), p.dispatch.adjust_logits(wide[:, 0].contiguous(), h.contiguous(), None, r))


def test_more_biases_and_history_than_share_a_word():
    p = pkg()
    g = torch.Generator(device="cuda").manual_seed(1)
    for n, m in ((1 << 20, 3), (50, 5000), (1 << 20, 5000)):
        logits = torch.randn(1, 9000, generator=g, device="cuda")
        h = torch.randint(0, 9000, (1, n), generator=g, device="cuda", dtype=torch.int32)
        h[:, ::2] = 8191   # more than a few bits of count
        ids = torch.randint(0, 9000, (1, m), generator=g, device="cuda", dtype=torch.int32)
        v, r = torch.randn(1, m, generator=g, device="cuda"), torch.tensor([[1.2, 0.3, 0.001]], device="cuda")
        agree(p.dispatch.adjust_logits(logits, h, None, r, ids, v), *expected(logits, h, None, r, ids, v))


def test_recorded_and_replayed():
    p = pkg()
    logits, h = torch.randn(2, 5000, device="cuda"), torch.zeros(2, 40, dtype=torch.int32, device="cuda")
    n, r, out = torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([[1.3, 0.2, 0.1]] * 2, device="cuda"), torch.empty(2, 5000, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        p.dispatch.adjust_logits(logits, h, n, r, out=out)
    for length in (0, 7, 40):
        n.fill_(length)
        h.random_(0, 5000)
        logits.normal_()
        g.replay()
        agree(out, *expected(logits, h, n, r))


def test_refusals():
    p = pkg()
    z, h, r = torch.zeros(2, 100, device="cuda"), torch.zeros(2, 5, dtype=torch.int32, device="cuda"), torch.ones(2, 3, device="cuda")
    ids, v = torch.zeros(2, 3, dtype=torch.int32, device="cuda"), torch.zeros(2, 3, device="cuda")
    for kw in (dict(logits=z.cpu()), dict(logits=z[0]), dict(logits=z.double()), dict(history=h), dict(rules=r), dict(history=h.long(), rules=r), dict(history=h[:1], rules=r),
               dict(history=h, rules=r[:1]), dict(history=h, rules=r.double()), dict(history=h, rules=r, lengths=h[:, 0].long()), dict(bias_ids=ids), dict(bias_ids=ids, bias_values=v[:1]),
               dict(bias_ids=ids.long(), bias_values=v), dict(allowed=torch.zeros(2, 3, dtype=torch.int32, device="cuda")), dict(allowed=torch.zeros(2, 4, device="cuda")),
               dict(out=z[:1]), dict(out=z.half()), dict(out=torch.zeros(2, 200, device="cuda")[:, ::2])):
        with pytest.raises(p.Ab2Error):
            p.dispatch.adjust_logits(**{"logits": z, **kw})
    assert p.dispatch.adjust_logits(z[:0]).shape == (0, 100)
    assert torch.equal(p.dispatch.adjust_logits(z, h[:, :0], None, r), z)
