"""Operators of a serving step over long contexts, as cases that can be timed and checked.

* ``append8``: new keys (rotated) and values of a ragged batch into pages of 8 bits, the queries rotated beside them.
* ``attention``: a ragged batch of new tokens attending to a paged cache of 8 bits, or to one of the queries' own type through a sliding
  window with a few first tokens that stay visible (sinks), or both.
* ``sample``: a token of every row of logits by temperature, top-k, top-p and min-p, from given random numbers.

Pages are [pages][kv heads][page size][head dim]; ``table`` [rows, pages a row may have] names a row's pages in order, ``lens``
its tokens with the new ones, ``starts`` where its new tokens begin in q, k and v.  Pages of 8 bits hold e4m3 numbers with a power of two for every 16 tokens
of a head: a value is its code times its block's scale.  Head counts are those of the dense classes and the layer stacks of this repository, windows and vocabularies theirs too.
"""
import importlib
import math
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
HEADS = [(32, 8, 128), (16, 4, 128), (32, 4, 128), (8, 8, 128), (16, 4, 64), (6, 2, 64)]
VOCABS = [8192, 32000, 128256]
BASE = 10000.0
BLOCK = 16          # tokens that share a scale
LARGEST = 448.0     # of e4m3
LEAST = -118        # the smallest exponent of a scale


def listed():
    return [
        # a decode step of a served batch into a cache of 8 bits
        dict(name="append8_step_64", op="append8", rows=64, new=1, ctx=500, heads=32, kv_heads=8, dim=128, rot=128, page=16, layout="half", dtype="bf16"),
        # prompts of several sessions in one pass, partly rotated heads, odd lengths
        dict(name="append8_prompt_5", op="append8", rows=5, new=2001, ctx=700, heads=16, kv_heads=4, dim=128, rot=64, page=64, layout="interleaved", dtype="bf16"),
        # one user: what a step costs in latency
        dict(name="attention8_step_1", op="attention", rows=1, new=1, ctx=700, heads=32, kv_heads=8, dim=128, page=16, pages="e4m3", window=0, sinks=0, dtype="bf16"),
        # a served batch of ragged sequences
        dict(name="attention8_step_48", op="attention", rows=48, new=1, ctx=8192, heads=32, kv_heads=8, dim=128, page=64, pages="e4m3", window=0, sinks=0, dtype="bf16"),
        # portions of prompts and single tokens of sessions in one pass
        dict(name="attention8_mixed_6", op="attention", rows=6, new=512, ctx=5000, heads=32, kv_heads=8, dim=128, page=32, pages="e4m3", window=0, sinks=0, dtype="bf16"),
        # a long document, a portion behind three
        dict(name="attention8_prompt_4096", op="attention", rows=1, new=4096, ctx=12288, heads=32, kv_heads=8, dim=128, page=128, pages="e4m3", window=0, sinks=0, dtype="bf16"),
        # sessions that have run for long, each seeing its last tokens and its first
        dict(name="window_step_32", op="attention", rows=32, new=1, ctx=30000, heads=32, kv_heads=8, dim=128, page=64, pages="own", window=2048, sinks=4, dtype="bf16"),
        # the same held in 8 bits, more sessions of a smaller class
        dict(name="window8_step_64", op="attention", rows=64, new=1, ctx=12000, heads=16, kv_heads=4, dim=128, page=16, pages="e4m3", window=1024, sinks=4, dtype="bf16"),
        # a long document read through a window
        dict(name="window_prompt_8000", op="attention", rows=1, new=8000, ctx=5000, heads=16, kv_heads=4, dim=128, page=64, pages="own", window=1024, sinks=4, dtype="bf16"),
        # the small f32 class reads a few prompts through a window
        dict(name="window_f32_chunk", op="attention", rows=3, new=130, ctx=380, heads=6, kv_heads=2, dim=64, page=16, pages="own", window=100, sinks=5, dtype="f32"),
        # a few sessions
        dict(name="sample_4", op="sample", rows=4, vocab=32000, dtype="f32"),
        # a large served batch with a large vocabulary
        dict(name="sample_64", op="sample", rows=64, vocab=128256, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["append8", "attention", "attention", "attention", "attention", "sample", "sample"])
    heads, kv_heads, dim = rng.choice(HEADS)
    if op == "sample":
        rows, vocab = _log(rng, 1, 64), rng.choice(VOCABS + [_log(rng, 50, 128256)])
        return dict(op=op, rows=rows, vocab=vocab, dtype="bf16" if rows * vocab > 4e6 else rng.choice(["bf16", "f32"]))
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "append8":
        rows = _log(rng, 1, 64)
        return dict(op=op, rows=rows, new=rng.choice([1, _log(rng, 1, 4096 // rows)]), ctx=_log(rng, 1, 32000 // rows), heads=heads, kv_heads=kv_heads, dim=dim,
                    rot=rng.choice([dim, dim, dim // 2, 24]), page=page, layout=rng.choice(["half", "interleaved"]), dtype="bf16")
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    pages = rng.choice(["e4m3", "e4m3", "own"])
    window = _log(rng, 16, 8192) if pages == "own" or rng.random() < 0.4 else 0
    sinks = rng.choice([0, 1, 4, _log(rng, 1, 300)]) if window else 0
    if rng.random() < 0.5:   # steps of single tokens
        rows = _log(rng, 1, 64)
        new, ctx = 1, _log(rng, 1, min(131072, 400000 // rows))
    else:                    # chunks; the scores of all rows stay below 2^29
        rows = rng.choice([1, 1, 2, 3, 5, 8])
        new = _log(rng, 2, 2048)
        ctx = _log(rng, 1, min(16384, max(1, (1 << 29) // (rows * heads * new) - new)))
        if dtype == "f32":
            new, ctx = min(new, 500), min(ctx, 2000)
    return dict(op=op, rows=rows, new=new, ctx=ctx, heads=heads, kv_heads=kv_heads, dim=dim, page=page, pages=pages, window=window, sinks=sinks, dtype=dtype)


def _lengths(case):
    """New tokens of every row and tokens before them: the first row has the most of both, the others less, single ones among them."""
    i = torch.arange(case["rows"], dtype=torch.float64)
    new = (case["new"] * (0.618034 * i % 1)).long().clamp(min=1)
    new[2::3] = 1
    ctx = (case["ctx"] * (0.25 + 0.75 * (0.754878 * i % 1))).long()
    new[0], ctx[0] = case["new"], case["ctx"]
    return new, ctx


def _powers(amax):
    """The least power of two with which amax, divided by it, is at most 448 = 0.875 * 2^9."""
    m, e = torch.frexp(amax)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, (e - 9 + (m > LARGEST / 512).int()), LEAST).clamp(min=LEAST))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = dict(case=case)
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        z = normal(rows, vocab, dtype=torch.float32) * 2.5
        likely = torch.randint(0, vocab, (rows, 32), generator=g, device="cuda")   # a text allows a few tokens well
        s["logits"] = z.scatter_add_(1, likely, 9 * uniform(rows, 32)).to(dt)
        s["uniforms"] = uniform(rows)
        s["temperature"] = 0.5 + 0.8 * uniform(rows)
        kind = torch.arange(rows, device="cuda")
        s["top_k"] = torch.where(kind % 4 == 1, 0, torch.exp(uniform(rows) * 5.5).int())     # 1 to 244, every fourth row without
        s["top_p"] = torch.where(kind % 5 == 3, torch.ones((), device="cuda"), 0.7 + 0.29 * uniform(rows))
        s["min_p"] = torch.where(kind % 3 == 2, 0.1 * uniform(rows), torch.zeros((), device="cuda"))
        return s
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    new, ctx = _lengths(case)
    rows, page = case["rows"], case["page"]
    lens = new + ctx
    need = (lens + page - 1) // page
    pages, most = int(need.sum()) + 8, int(need.max()) + 2
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)   # sessions came and went: pages lie anywhere
    ends = torch.cumsum(need, 0)
    at = torch.arange(most)[None, :] + (ends - need)[:, None]
    inside = torch.arange(most)[None, :] < need[:, None]
    s["table"] = torch.where(inside.cuda(), order[at.clamp(max=pages - 1).cuda()], torch.zeros((), dtype=torch.int32, device="cuda")).contiguous()
    s["lens"] = lens.to(torch.int32).cuda()
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(new, 0)])
    s["starts"] = None if case["new"] == 1 else starts.to(torch.int32).cuda()
    T = int(starts[-1])
    s["max_new"] = int(new.max())
    louder = 1 + 3 * (torch.rand(kv_heads, 1, dim, generator=g, device="cuda") < 0.03).to(dt)   # a few dimensions of keys are larger than the others
    s["k_pages"], s["v_pages"] = normal(pages, kv_heads, page, dim) * louder, normal(pages, kv_heads, page, dim)
    s["k_scales"] = s["v_scales"] = None
    if case["op"] == "append8" or case["pages"] == "e4m3":
        for n in ("k", "v"):
            x = s[n + "_pages"].float().view(pages, kv_heads, page // BLOCK, BLOCK * dim)
            scale = _powers(x.abs().amax(-1))
            if case["op"] == "append8":   # what blocks held before: some smaller, some larger than the new tokens need
                scale = scale * torch.exp2(torch.randint(-1, 2, scale.shape, generator=g, device="cuda").float())
                x = x.clamp(-LARGEST * scale[..., None], LARGEST * scale[..., None])
            s[n + "_pages"] = (x / scale[..., None]).to(torch.float8_e4m3fn).view(pages, kv_heads, page, dim)
            s[n + "_scales"] = scale
    s["q"] = normal(T, heads, dim)
    if case["op"] == "append8":
        s["k"], s["v"] = normal(T, kv_heads, dim) * louder.view(kv_heads, dim), normal(T, kv_heads, dim)
        s["frequencies"] = BASE ** (-2.0 * torch.arange(case["rot"] // 2, dtype=torch.float64, device="cuda") / case["rot"])
    else:
        s["q"] = s["q"] * 2   # a softmax that tells keys apart
        s["scale"] = 1.0 / math.sqrt(dim)
        s["longest"] = int(lens.max())
    return s


# -- plain forms ---------------------------------------------------------------------------------------

def _rotated(x, positions, f, layout):
    a = positions.double()[:, None] * f
    c, s = a.cos().float()[:, None, :], a.sin().float()[:, None, :]
    n, xf = f.numel(), x.float()
    if layout == "half":
        x1, x2 = xf[..., :n], xf[..., n:2 * n]
        turned = torch.cat([x1 * c - x2 * s, x1 * s + x2 * c], dim=-1)
    else:
        x1, x2 = xf[..., 0:2 * n:2], xf[..., 1:2 * n:2]
        turned = torch.stack([x1 * c - x2 * s, x1 * s + x2 * c], dim=-1).flatten(-2)
    return torch.cat([turned, xf[..., 2 * n:]], dim=-1).to(x.dtype)


def _rows_of(s):
    """Row and position of every new token."""
    rows = s["lens"].numel()
    if s["starts"] is None:
        return torch.arange(rows, device="cuda"), s["lens"].long() - 1
    starts = s["starts"].long()
    t = torch.arange(s["q"].shape[0], device="cuda")
    row = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    return row, s["lens"].long()[row] - starts[row + 1] + t


def _put(x, pages, scales, where, slot):
    """x [tokens, kv_heads, dim] into slots of pages, whose blocks' scales grow where they have to."""
    P, kv, per = scales.shape
    dim, T = x.shape[-1], x.shape[0]
    x = x.float()
    block = where * per + slot // BLOCK
    amax = torch.where(x.isfinite(), x.abs(), torch.zeros((), device="cuda")).amax(-1)
    top = torch.zeros(P * per, kv, device="cuda").scatter_reduce_(0, block[:, None].expand(T, kv), amax, "amax")[block]   # of the token's block
    first = torch.full((P * per,), BLOCK, device="cuda").scatter_reduce_(0, block, slot % BLOCK, "amin")[block]            # the block's first new slot
    old = torch.where(first[:, None] == 0, torch.zeros((), device="cuda"), scales[where, :, slot // BLOCK])
    scale = torch.maximum(_powers(top), old)
    bytes_ = pages.view(torch.uint8).view(P, kv, per, BLOCK, dim)
    there = bytes_[where, :, slot // BLOCK]                                                                                # [tokens, kv, 16, dim]
    held = (there.view(torch.float8_e4m3fn).float() * (old / scale)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    earlier = torch.arange(BLOCK, device="cuda")[None, None, :, None] < first[:, None, None, None]
    bytes_[where, :, slot // BLOCK] = torch.where(earlier, held, there)
    bytes_[where, :, slot // BLOCK, slot % BLOCK] = (x / scale[..., None]).to(torch.float8_e4m3fn).view(torch.uint8)
    scales[where, :, slot // BLOCK] = scale


def _plain_append(s):
    case = s["case"]
    row, pos = _rows_of(s)
    page = case["page"]
    where, slot = s["table"].long()[row, pos // page], pos % page
    _put(_rotated(s["k"], pos, s["frequencies"], case["layout"]), s["k_pages"], s["k_scales"], where, slot)
    _put(s["v"], s["v_pages"], s["v_scales"], where, slot)
    return _rotated(s["q"], pos, s["frequencies"], case["layout"]), s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]


def _plain_attention(s):
    case = s["case"]
    rows, heads, kv_heads, dim = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    n, L, page = s["max_new"], s["longest"], case["page"]
    row, pos = _rows_of(s)
    used = (L + page - 1) // page
    at = s["table"][:, :used].long()

    def gathered(name):   # [rows, kv_heads, 1, keys, dim]
        p, scales = s[name + "_pages"], s[name + "_scales"]
        if scales is None:
            x = p[at].float()
        else:
            x = p.view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * scales[at].repeat_interleave(BLOCK, dim=-1)[..., None]
        return x.permute(0, 2, 1, 3, 4).reshape(rows, kv_heads, 1, used * page, dim)[:, :, :, :L]

    # every row's new tokens, the last of them at the end of n places
    place = n - s["lens"].long()[row] + pos
    q = torch.zeros(rows, n, heads, dim, device="cuda")
    q[row, place] = s["q"].float()
    q = q.view(rows, n, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    w = torch.matmul(q * s["scale"], gathered("k").transpose(-1, -2))
    last = (s["lens"].long()[:, None] - n + torch.arange(n, device="cuda")[None, :])[:, :, None]
    j = torch.arange(L, device="cuda")[None, None, :]
    seen = j <= last
    if case["window"]:
        seen = seen & ((last - j < case["window"]) | (j < case["sinks"]))
    w.masked_fill_(~seen[:, None, None], -torch.inf)
    w -= w.amax(-1, keepdim=True).clamp(min=-1e30)
    w.exp_()
    total = w.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(w, gathered("v")) / total
    return o.permute(0, 3, 1, 2, 4).reshape(rows, n, heads, dim)[row, place].to(s["q"].dtype)


def _plain_sample(s):
    z = s["logits"].double() / s["temperature"].double()[:, None]
    rows, vocab = z.shape
    z, order = torch.sort(z, dim=1, descending=True, stable=True)   # equal ones: the lower index first
    p = torch.exp(z - z[:, :1])
    k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
    p = torch.where(torch.arange(vocab, device="cuda")[None, :] < k, p, 0.0)
    before = torch.cumsum(p, dim=1) - p
    keep = (before < s["top_p"].double()[:, None] * p.sum(1, keepdim=True)) & (p >= s["min_p"].double()[:, None])
    keep[:, 0] = True
    p = torch.zeros_like(p).scatter_(1, order, torch.where(keep, p, 0.0))
    up = torch.cumsum(p, dim=1)
    return (up <= s["uniforms"].double()[:, None] * up[:, -1:]).sum(1).to(torch.int32)


def run(s):
    case = s["case"]
    if own:
        ops = _package().dispatch
        if case["op"] == "sample":
            return ops.sample(s["logits"], s["uniforms"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        scales = None if s["k_scales"] is None else (s["k_scales"], s["v_scales"])
        if case["op"] == "append8":
            q = ops.paged_append(s["k_pages"], s["v_pages"], s["k"], s["v"], s["table"], s["lens"], s["starts"], q=s["q"],
                                 frequencies=s["frequencies"], layout=case["layout"], scales=scales)
            return q, s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"]
        return ops.attention_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["scale"], s["starts"], s["max_new"],
                                   scales=scales, window=case["window"], sinks=case["sinks"])
    return {"append8": _plain_append, "attention": _plain_attention, "sample": _plain_sample}[case["op"]](s)


def _package():
    name = "aarambh_ai_b200"
    if name not in sys.modules:
        importlib.import_module("__graft_entry__").import_package()
    return sys.modules[name]


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * 24, "flops": 4 * n}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    new, ctx = (v.tolist() for v in _lengths(case))
    T = sum(new)
    if case["op"] == "append8":
        return {"bytes": 2 * T * heads * dim * size + 2 * T * kv_heads * dim * (size + 1), "flops": 3 * T * (heads + kv_heads) * case["rot"] + 4 * T * kv_heads * dim}
    W, first = case["window"] or 1 << 40, case["sinks"]

    def visible(n):   # the sum over lengths 1 .. n of the keys that the last token sees: min(length, W + sinks)
        m = min(n, W + first)
        return m * (m + 1) / 2 + (n - m) * m

    keys = sum(min(c + n, n + W - 1 + first) for n, c in zip(new, ctx))
    scores = sum(visible(c + n) - visible(c) for n, c in zip(new, ctx))
    each = dim + 4 / BLOCK if case["pages"] == "e4m3" else dim * size
    return {"bytes": 2 * keys * kv_heads * each + 2 * T * heads * dim * size, "flops": 4 * scores * heads * dim}


# -- the definitions in 64 bits ------------------------------------------------------------------------

def _turned(x, positions, f, layout):
    """Pairs as complex numbers times e^(i angle)."""
    n = f.numel()
    x = x.double()
    pairs = torch.complex(x[..., :n], x[..., n:2 * n]) if layout == "half" else torch.view_as_complex(x[..., :2 * n].reshape(*x.shape[:-1], n, 2).contiguous())
    angle = torch.outer(positions.double(), f)
    y = pairs * torch.polar(torch.ones_like(angle), angle)[:, None, :]
    out = x.clone()
    if layout == "half":
        out[..., :n], out[..., n:2 * n] = y.real, y.imag
    else:
        out[..., :2 * n] = torch.view_as_real(y).flatten(-2)
    return out


def _chosen(z, u, T, k, p, least):
    """One row's token: a loop over what is kept, the likeliest first."""
    z = z.double() / T
    w = torch.exp(z - z.max())
    order = torch.argsort(-z, stable=True)[:k if k > 0 else z.numel()]
    up = torch.cumsum(w[order], 0)
    m = max(1, min(int(torch.searchsorted(up, p * up[-1])) + 1 if p < 1 else len(order), int((w[order] >= least).sum())))
    kept = torch.sort(order[:m])[0]
    up = torch.cumsum(w[kept], 0)
    return int(kept[min(int(torch.searchsorted(up, u * up[-1], right=True)), m - 1)])


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        rules = [s[n].double().tolist() for n in ("uniforms", "temperature", "top_k", "top_p", "min_p")]
        return torch.tensor([_chosen(s["logits"][r], u, t, int(k), p, m) for r, (u, t, k, p, m) in enumerate(zip(*rules))], dtype=torch.int32)
    page, rows = case["page"], case["rows"]
    starts = list(range(rows + 1)) if s["starts"] is None else s["starts"].tolist()
    lens = s["lens"].tolist()
    if case["op"] == "append8":
        q, pools = [], {n: (s[n + "_pages"].double(), s[n + "_scales"].double()) for n in ("k", "v")}
        table = s["table"].tolist()
        for r in range(rows):
            a, b = starts[r], starts[r + 1]
            pos = torch.arange(lens[r] - (b - a), lens[r], device="cuda")
            q.append(_turned(s["q"][a:b], pos, s["frequencies"], case["layout"]))
            for n, (codes, scales) in pools.items():
                x = _turned(s["k"][a:b], pos, s["frequencies"], case["layout"]).to(s["k"].dtype).double() if n == "k" else s["v"][a:b].double()
                first = lens[r] - (b - a)
                for block in range(first // BLOCK, (lens[r] - 1) // BLOCK + 1):
                    lo, hi = max(first, block * BLOCK), min(lens[r], (block + 1) * BLOCK)
                    here, at, i = table[r][block * BLOCK // page], block * BLOCK % page, block * BLOCK % page // BLOCK
                    y = x[lo - first:hi - first]
                    # a largest value of 448 times a power of two needs that power, and its logarithm comes out a little above it
                    scale = torch.exp2(torch.ceil(torch.log2(y.abs().amax((0, 2)) / LARGEST) - 1e-9).clamp(min=LEAST))
                    if lo > block * BLOCK:
                        old = scales[here, :, i].clone()
                        scale = torch.maximum(scale, old)
                        codes[here, :, at:at + lo % BLOCK] *= (old / scale)[:, None, None]
                    codes[here, :, at + lo % BLOCK:at + lo % BLOCK + hi - lo] = (y / scale[None, :, None]).transpose(0, 1)
                    scales[here, :, i] = scale
        return torch.cat(q), pools["k"][0], pools["v"][0], pools["k"][1], pools["v"][1]
    group = case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for r in range(rows):
        a, b, L = starts[r], starts[r + 1], lens[r]
        ids = s["table"][r, :(L + page - 1) // page].long()
        back = torch.arange(L - (b - a), L, device="cuda")[:, None] - torch.arange(L, device="cuda")[None, :]
        hidden = back < 0
        if case["window"]:
            hidden = hidden | ((back >= case["window"]) & (torch.arange(L, device="cuda")[None, :] >= case["sinks"]))
        for head in range(case["kv_heads"]):
            kv = []
            for n in ("k", "v"):
                x = s[n + "_pages"].view(torch.uint8 if case["pages"] == "e4m3" else s["q"].dtype)[ids, head]
                if case["pages"] == "e4m3":
                    x = x.view(torch.float8_e4m3fn).double().unflatten(1, (-1, BLOCK)) * s[n + "_scales"][ids, head].double()[..., None, None]
                kv.append(x.reshape(-1, case["dim"])[:L].double())
            for h in range(head * group, (head + 1) * group):
                x = s["scale"] * (s["q"][a:b, h].double() @ kv[0].T)
                out[a:b, h] = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1) @ kv[1]
    return out
