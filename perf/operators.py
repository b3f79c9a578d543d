"""Four operators of a serving step, as cases that can be timed and checked.

* ``rotary``: q and k of a batch of tokens rotated by their positions.
* ``append``: new keys (rotated) and values of a ragged batch into the pages of a cache, the queries rotated beside them.
* ``attention``: a ragged batch of new tokens, single ones or chunks, attending to a paged cache.
* ``logits``: penalties for repeated tokens, biases and a grammar's mask on the logits of a batch.

Pages are [pages][kv heads][page size][head dim]; ``table`` [rows, pages a row may have] names a row's pages in order, ``lens``
its tokens with the new ones, ``starts`` where its new tokens begin in q, k and v.  Head counts are those of the dense classes
and the layer stacks of this repository, vocabularies theirs too.
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
RAMP = dict(factor=4.0, original=8192, low=1.0, high=32.0)   # a context four times as long as the one learnt
RAMP_MAGNITUDE = 0.1 * math.log(RAMP["factor"]) + 1.0


def listed():
    return [
        # one step of a few sessions far into long conversations: latency
        dict(name="rotary_step_8", op="rotary", tokens=8, heads=32, kv_heads=8, dim=128, rot=128, layout="half", scaled=False, dtype="bf16", first=90000),
        # a partly rotated head of the small f32 class, odd token count
        dict(name="rotary_part_1777", op="rotary", tokens=1777, heads=6, kv_heads=2, dim=64, rot=24, layout="interleaved", scaled=False, dtype="f32", first=0),
        # a long document's portion behind what a scaled model has read already
        dict(name="rotary_prompt_8192", op="rotary", tokens=8192, heads=32, kv_heads=8, dim=128, rot=128, layout="half", scaled=True, dtype="bf16", first=20000),
        # a decode step of a served batch
        dict(name="append_step_64", op="append", rows=64, new=1, ctx=500, heads=32, kv_heads=8, dim=128, page=16, layout="half", scaled=False, dtype="bf16"),
        # prompts of several sessions in one pass
        dict(name="append_prompt_5", op="append", rows=5, new=2001, ctx=700, heads=16, kv_heads=4, dim=128, page=64, layout="interleaved", scaled=True, dtype="bf16"),
        # one user: what a step costs in latency
        dict(name="attention_step_1", op="attention", rows=1, new=1, ctx=700, heads=32, kv_heads=8, dim=128, page=16, dtype="bf16"),
        # a served batch of ragged sequences
        dict(name="attention_step_48", op="attention", rows=48, new=1, ctx=8192, heads=32, kv_heads=8, dim=128, page=64, dtype="bf16"),
        # the small f32 class reads a few prompts
        dict(name="attention_f32_chunk", op="attention", rows=3, new=130, ctx=380, heads=6, kv_heads=2, dim=64, page=16, dtype="f32"),
        # portions of prompts and single tokens of sessions in one pass
        dict(name="attention_mixed_6", op="attention", rows=6, new=512, ctx=5000, heads=32, kv_heads=8, dim=128, page=32, dtype="bf16"),
        # a long document, a portion behind three
        dict(name="attention_prompt_4096", op="attention", rows=1, new=4096, ctx=12288, heads=32, kv_heads=8, dim=128, page=128, dtype="bf16"),
        # a few sessions with rules
        dict(name="logits_4", op="logits", rows=4, vocab=32000, history=300, biases=20, masked=True, dtype="f32"),
        # a large served batch with a large vocabulary and long histories
        dict(name="logits_64", op="logits", rows=64, vocab=128256, history=4096, biases=300, masked=True, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attention", "attention", "attention", "logits"])
    heads, kv_heads, dim = rng.choice(HEADS)
    if op == "rotary":
        rot = rng.choice([dim, dim, dim // 2, 24])
        return dict(op=op, tokens=_log(rng, 1, 8192), heads=heads, kv_heads=kv_heads, dim=dim, rot=rot, layout=rng.choice(["half", "interleaved"]),
                    scaled=rng.random() < 0.4, dtype=rng.choice(["bf16", "bf16", "f32"]) if heads < 32 else "bf16", first=rng.randint(0, 100000))
    if op == "append":
        rows = _log(rng, 1, 64)
        return dict(op=op, rows=rows, new=rng.choice([1, _log(rng, 1, 4096 // rows)]), ctx=_log(rng, 1, 32000 // rows), heads=heads, kv_heads=kv_heads, dim=dim,
                    page=rng.choice([16, 32, 64, 128, 256]), layout=rng.choice(["half", "interleaved"]), scaled=rng.random() < 0.4,
                    dtype=rng.choice(["bf16", "bf16", "f32"]))
    if op == "logits":
        rows, vocab = _log(rng, 1, 64), rng.choice(VOCABS)
        return dict(op=op, rows=rows, vocab=vocab, history=_log(rng, 1, 4096), biases=rng.choice([0, 1, _log(rng, 1, 300)]), masked=rng.random() < 0.6,
                    dtype="bf16" if rows * vocab > 4e6 else rng.choice(["bf16", "f32"]))
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if rng.random() < 0.5:   # steps of single tokens
        rows = _log(rng, 1, 64)
        new, ctx = 1, _log(rng, 1, min(131072, 400000 // rows))
    else:                    # chunks; the scores of all rows stay below 2^29
        rows = rng.choice([1, 1, 2, 3, 5, 8])
        new = _log(rng, 2, 2048)
        ctx = _log(rng, 1, min(16384, max(1, (1 << 29) // (rows * heads * new) - new)))
        if dtype == "f32":
            new, ctx = min(new, 500), min(ctx, 2000)
    return dict(op=op, rows=rows, new=new, ctx=ctx, heads=heads, kv_heads=kv_heads, dim=dim, page=rng.choice([16, 32, 64, 128, 256]), dtype=dtype)


def _lengths(case):
    """New tokens of every row and tokens before them: the first row has the most of both, the others less, single ones among them."""
    i = torch.arange(case["rows"], dtype=torch.float64)
    new = (case["new"] * (0.618034 * i % 1)).long().clamp(min=1)
    new[2::3] = 1
    ctx = (case["ctx"] * (0.25 + 0.75 * (0.754878 * i % 1))).long()
    new[0], ctx[0] = case["new"], case["ctx"]
    return new, ctx


def _frequencies(case):
    """Radians a position turns each pair by (f64), and what multiplies the rotated pairs."""
    rot = case.get("rot", case["dim"])
    f = BASE ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
    if not case["scaled"]:
        return f, 1.0
    turns = RAMP["original"] * f / (2 * math.pi)
    keep = ((turns - RAMP["low"]) / (RAMP["high"] - RAMP["low"])).clamp(0, 1)
    return f / RAMP["factor"] * (1 - keep) + f * keep, RAMP_MAGNITUDE


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape, dtype=dt):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dtype)

    s = dict(case=case)
    if case["op"] == "logits":
        rows, vocab, n = case["rows"], case["vocab"], case["history"]
        s["logits"] = normal(rows, vocab) * 3
        # text repeats itself: half of a history comes from a small part of the vocabulary
        some, all_ = (torch.randint(0, m, (rows, n), generator=g, device="cuda", dtype=torch.int32) for m in (64, vocab))
        s["history"] = torch.where(torch.rand(rows, n, generator=g, device="cuda") < 0.5, some * (vocab // 64), all_)
        s["lengths"] = torch.randint(n // 2, n + 1, (rows,), generator=g, device="cuda", dtype=torch.int32)
        r = torch.rand(rows, 3, generator=g, device="cuda")
        s["rules"] = torch.stack([1.0 + 0.5 * r[:, 0], r[:, 1], 0.3 * r[:, 2]], dim=1).contiguous()  # repetition, presence, frequency
        s["bias_ids"] = s["bias_values"] = s["allowed"] = None
        if case["biases"]:
            s["bias_ids"] = torch.stack([torch.randperm(vocab, generator=g, device="cuda")[:case["biases"]] for _ in range(rows)]).to(torch.int32)
            s["bias_values"] = normal(rows, case["biases"], dtype=torch.float32) * 4
        if case["masked"]:
            words = (vocab + 31) // 32
            a, b = (torch.randint(-2 ** 31, 2 ** 31, (rows, words), generator=g, device="cuda", dtype=torch.int64) for _ in range(2))
            s["allowed"] = (a | b).to(torch.int32)   # three of four tokens
        return s
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] != "attention":
        f, s["magnitude"] = _frequencies(case)
        s["frequencies"] = f.cuda()
    if case["op"] == "rotary":
        T = case["tokens"]
        s["q"], s["k"] = normal(T, heads, dim), normal(T, kv_heads, dim)
        s["positions"] = (case["first"] + torch.arange(T, device="cuda")).to(torch.int32)
        return s
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
    s["k_pages"], s["v_pages"] = (normal(pages, kv_heads, page, dim) for _ in range(2))
    s["q"] = normal(T, heads, dim)
    if case["op"] == "append":
        s["k"], s["v"] = normal(T, kv_heads, dim), normal(T, kv_heads, dim)
    else:
        s["q"] = s["q"] * 2   # a softmax that tells keys apart
        s["scale"] = 1.0 / math.sqrt(dim)
        s["longest"] = int(lens.max())
    return s


# -- plain forms ---------------------------------------------------------------------------------------

def _rotated(x, positions, f, magnitude, layout):
    a = positions.double()[:, None] * f
    c, s = (a.cos() * magnitude).float()[:, None, :], (a.sin() * magnitude).float()[:, None, :]
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


def _plain_append(s):
    case = s["case"]
    row, pos = _rows_of(s)
    page = case["page"]
    where, slot = s["table"].long()[row, pos // page], pos % page
    s["k_pages"][where, :, slot] = _rotated(s["k"], pos, s["frequencies"], s["magnitude"], case["layout"])
    s["v_pages"][where, :, slot] = s["v"]
    return _rotated(s["q"], pos, s["frequencies"], s["magnitude"], case["layout"]), s["k_pages"], s["v_pages"]


def _plain_attention(s):
    case = s["case"]
    rows, heads, kv_heads, dim = case["rows"], case["heads"], case["kv_heads"], case["dim"]
    n, L, page = s["max_new"], s["longest"], case["page"]
    row, pos = _rows_of(s)
    used = (L + page - 1) // page
    at = s["table"][:, :used].long()

    def gathered(p):   # [rows, kv_heads, 1, keys, dim]
        return p[at].permute(0, 2, 1, 3, 4).reshape(rows, kv_heads, 1, used * page, dim)[:, :, :, :L].float()

    # every row's new tokens, the last of them at the end of n places
    place = n - s["lens"].long()[row] + pos
    q = torch.zeros(rows, n, heads, dim, device="cuda")
    q[row, place] = s["q"].float()
    q = q.view(rows, n, kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    w = torch.matmul(q * s["scale"], gathered(s["k_pages"]).transpose(-1, -2))
    last = s["lens"].long()[:, None] - n + torch.arange(n, device="cuda")[None, :]
    seen = torch.arange(L, device="cuda")[None, None, :] <= last[:, :, None]
    w.masked_fill_(~seen[:, None, None], -torch.inf)
    w -= w.amax(-1, keepdim=True).clamp(min=-1e30)
    w.exp_()
    total = w.sum(-1, keepdim=True).clamp(min=1e-30)
    o = torch.matmul(w, gathered(s["v_pages"])) / total
    return o.permute(0, 3, 1, 2, 4).reshape(rows, n, heads, dim)[row, place].to(s["q"].dtype)


def _plain_logits(s):
    z = s["logits"].float()
    rows, vocab = z.shape
    inside = torch.arange(s["history"].shape[1], device="cuda")[None, :] < s["lengths"][:, None]
    count = torch.zeros(rows, vocab, device="cuda").scatter_add_(1, s["history"].long(), inside.float())
    rho, presence, frequency = (s["rules"][:, i:i + 1] for i in range(3))
    z = torch.where(count > 0, torch.where(z > 0, z / rho, z * rho) - (presence + frequency * count), z)
    if s["bias_ids"] is not None:   # a row's ids are distinct
        z = z + torch.zeros_like(z).scatter_(1, s["bias_ids"].long(), s["bias_values"])
    if s["allowed"] is not None:
        v = torch.arange(vocab, device="cuda")
        z = torch.where((s["allowed"][:, v >> 5] >> (v & 31)[None, :]) & 1 != 0, z, -torch.inf)
    return z.to(s["logits"].dtype)


def run(s):
    case = s["case"]
    if own:
        ops = _package().dispatch
        if case["op"] == "rotary":
            return ops.rotary_apply(s["q"], s["k"], s["positions"], s["frequencies"], case["layout"], s["magnitude"])
        if case["op"] == "append":
            q = ops.paged_append(s["k_pages"], s["v_pages"], s["k"], s["v"], s["table"], s["lens"], s["starts"], q=s["q"],
                                 frequencies=s["frequencies"], layout=case["layout"], magnitude=s["magnitude"])
            return q, s["k_pages"], s["v_pages"]
        if case["op"] == "attention":
            return ops.attention_paged(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], s["scale"], s["starts"], s["max_new"])
        return ops.adjust_logits(s["logits"], s["history"], s["lengths"], s["rules"], s["bias_ids"], s["bias_values"], s["allowed"])
    if case["op"] == "rotary":
        return tuple(_rotated(x, s["positions"], s["frequencies"], s["magnitude"], case["layout"]) for x in (s["q"], s["k"]))
    return {"append": _plain_append, "attention": _plain_attention, "logits": _plain_logits}[case["op"]](s)


def _package():
    name = "aarambh_ai_b200"
    if name not in sys.modules:
        importlib.import_module("__graft_entry__").import_package()
    return sys.modules[name]


def work(case):
    size = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "logits":
        n = case["rows"] * case["vocab"]
        return {"bytes": 2 * n * size + (n / 8 if case["masked"] else 0) + case["rows"] * (3 * case["history"] + 8 * case["biases"]), "flops": 4 * n}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "rotary":
        n = case["tokens"] * (heads + kv_heads)
        return {"bytes": 2 * n * dim * size, "flops": 3 * n * case["rot"]}
    new, ctx = (v.tolist() for v in _lengths(case))
    if case["op"] == "append":
        T = sum(new)
        return {"bytes": 2 * T * (heads + 2 * kv_heads) * dim * size, "flops": 3 * T * (heads + kv_heads) * dim}
    keys = sum(n + c for n, c in zip(new, ctx))
    scores = sum(n * c + n * (n + 1) / 2 for n, c in zip(new, ctx))
    return {"bytes": (2 * keys * kv_heads + 2 * sum(new) * heads) * dim * size, "flops": 4 * scores * heads * dim}


# -- the definitions in 64 bits ------------------------------------------------------------------------

def _turned(x, positions, f, magnitude, layout):
    """Pairs as complex numbers times magnitude e^(i angle)."""
    n = f.numel()
    x = x.double()
    pairs = torch.complex(x[..., :n], x[..., n:2 * n]) if layout == "half" else torch.view_as_complex(x[..., :2 * n].reshape(*x.shape[:-1], n, 2).contiguous())
    angle = torch.outer(positions.double(), f)
    y = pairs * torch.polar(torch.full_like(angle, magnitude), angle)[:, None, :]
    out = x.clone()
    if layout == "half":
        out[..., :n], out[..., n:2 * n] = y.real, y.imag
    else:
        out[..., :2 * n] = torch.view_as_real(y).flatten(-2)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return tuple(_turned(x, s["positions"], s["frequencies"], s["magnitude"], case["layout"]) for x in (s["q"], s["k"]))
    if case["op"] == "logits":
        z = s["logits"].double()
        rules = s["rules"].double()
        for r in range(case["rows"]):
            ids, count = torch.unique(s["history"][r, :int(s["lengths"][r])].long(), return_counts=True)
            old = z[r, ids]
            z[r, ids] = old * torch.where(old > 0, 1 / rules[r, 0], rules[r, 0]) - rules[r, 1] - rules[r, 2] * count
            if s["bias_ids"] is not None:
                z[r, s["bias_ids"][r].long()] += s["bias_values"][r].double()
            if s["allowed"] is not None:
                bits = (s["allowed"][r][:, None] & (1 << torch.arange(32, device="cuda"))).ne(0).flatten()[:case["vocab"]]
                z[r, ~bits] = -math.inf
        return z
    page, rows = case["page"], case["rows"]
    starts = list(range(rows + 1)) if s["starts"] is None else s["starts"].tolist()
    lens = s["lens"].tolist()
    if case["op"] == "append":
        kp, vp, q = s["k_pages"].double(), s["v_pages"].double(), []
        for r in range(rows):
            a, b = starts[r], starts[r + 1]
            pos = torch.arange(lens[r] - (b - a), lens[r], device="cuda")
            ids = s["table"][r].long()[torch.div(pos, page, rounding_mode="floor")]
            kp[ids, :, pos % page] = _turned(s["k"][a:b], pos, s["frequencies"], s["magnitude"], case["layout"])
            vp[ids, :, pos % page] = s["v"][a:b].double()
            q.append(_turned(s["q"][a:b], pos, s["frequencies"], s["magnitude"], case["layout"]))
        return torch.cat(q), kp, vp
    group = case["heads"] // case["kv_heads"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for r in range(rows):
        a, b, L = starts[r], starts[r + 1], lens[r]
        ids = s["table"][r, :(L + page - 1) // page].long()
        for h in range(case["heads"]):
            k, v = (p[ids, h // group].reshape(-1, case["dim"])[:L].double() for p in (s["k_pages"], s["v_pages"]))
            x = s["scale"] * (s["q"][a:b, h].double() @ k.T)
            late = torch.arange(L, device="cuda")[None, :] > torch.arange(L - (b - a), L, device="cuda")[:, None]
            out[a:b, h] = torch.softmax(x.masked_fill(late, -math.inf), dim=-1) @ v
    return out
