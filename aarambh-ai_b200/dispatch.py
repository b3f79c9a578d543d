"""Host-side mirror of the reference's kernel dispatch entry points
(crates/aarambh-studio-kernel/src/dispatch.rs): rms_norm, attention_forward_causal,
plus the fused RoPE / SwiGLU wrappers and the greedy argmax.  Outputs are freshly
allocated, inputs are borrowed, tensors must be CUDA and are made contiguous.
"""
from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import check, lib
from .qlinear import dtype_code, stream_ptr


def _cuda(t: torch.Tensor, what: str) -> torch.Tensor:
    if not t.is_cuda:
        raise _lib.Ab2Error(-7, f"{what} must be a CUDA tensor (this library has no CPU path)")
    return t.contiguous()


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    x = _cuda(x, "x")
    d = x.shape[-1] if x.dim() else 0
    if x.dim() < 1 or d == 0:
        raise _lib.Ab2Error(-1, "rms_norm hidden dimension must be non-zero")
    if tuple(weight.shape) != (d,):
        raise _lib.Ab2Error(-1, f"rms_norm weight must have shape [{d}], got {list(weight.shape)}")
    w = _cuda(weight, "weight").float()
    out = torch.empty_like(x)
    check(lib.ab2_rms_norm(x.data_ptr(), w.data_ptr(), out.data_ptr(), x.numel() // d, d, float(eps),
                           dtype_code(x.dtype), stream_ptr()))
    return out


def fused_rope_apply(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor, seqlen_offset: int) -> torch.Tensor:
    """x [batch, seq, heads, head_dim]; cos, sin [max_seq, head_dim/2] (f32)."""
    x = _cuda(x, "x")
    if x.dim() != 4:
        raise _lib.Ab2Error(-1, f"RoPE input must be [batch, seq, heads, head_dim], got {list(x.shape)}")
    b, s, h, hd = x.shape
    cos = _cuda(cos, "cos").float(); sin = _cuda(sin, "sin").float()
    if cos.shape != sin.shape or cos.dim() != 2 or cos.shape[1] * 2 != hd:
        raise _lib.Ab2Error(-1, "RoPE tables must be [max_seq, head_dim/2]")
    out = torch.empty_like(x)
    check(lib.ab2_rope_apply(x.data_ptr(), out.data_ptr(), cos.data_ptr(), sin.data_ptr(), b, s, h, hd,
                             seqlen_offset, cos.shape[0], dtype_code(x.dtype), stream_ptr()))
    return out


def fused_swiglu(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    if gate.shape != up.shape or gate.dtype != up.dtype:
        raise _lib.Ab2Error(-1, "SwiGLU gate and up must have the same shape and dtype")
    gate = _cuda(gate, "gate"); up = _cuda(up, "up")
    out = torch.empty_like(gate)
    check(lib.ab2_swiglu(gate.data_ptr(), up.data_ptr(), out.data_ptr(), gate.numel(), dtype_code(gate.dtype),
                         stream_ptr()))
    return out


def attention_forward_causal(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float) -> torch.Tensor:
    """q [b, h, q_len, hd]; k, v [b, kv_heads, kv_len, hd] (kv heads not repeated)."""
    q = _cuda(q, "q"); k = _cuda(k, "k"); v = _cuda(v, "v")
    if q.dim() != 4 or k.dim() != 4 or v.shape != k.shape:
        raise _lib.Ab2Error(-1, "attention expects rank-4 q and matching rank-4 k, v")
    if q.shape[0] != k.shape[0]:
        raise _lib.Ab2Error(-1, "attention batch dimensions must match")
    if q.shape[3] != k.shape[3]:
        raise _lib.Ab2Error(-1, "attention head dimensions must match")
    if q.dtype != k.dtype or q.dtype != v.dtype:
        raise _lib.Ab2Error(-3, "attention tensors must share one dtype")
    b, h, ql, hd = q.shape
    out = torch.empty_like(q)
    check(lib.ab2_attention_causal(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), b, h, k.shape[1],
                                   ql, k.shape[2], hd, float(scale), dtype_code(q.dtype), stream_ptr()))
    return out


def attention_decode(cache, q: torch.Tensor, scale: float, layer: int = 0, row0: int = 0) -> torch.Tensor:
    """q [rows, n_heads, head_dim]: one query per sequence over its cache."""
    q = _cuda(q, "q")
    out = torch.empty_like(q)
    check(lib.ab2_attention_decode(cache._h, layer, q.data_ptr(), out.data_ptr(), row0, q.shape[0],
                                   float(scale), dtype_code(q.dtype), stream_ptr()))
    return out


def attention_decode_static(cache, q: torch.Tensor, scale: float, out: torch.Tensor, layer: int = 0,
                            row0: int = 0) -> torch.Tensor:
    """``attention_decode`` for hosts that must not allocate on the device: the
    caller supplies ``out`` and the split scratch is a fixed array inside the
    library (8 MiB; larger problems are rejected).  Calls on different streams
    must not overlap."""
    if not q.is_contiguous() or not out.is_contiguous() or out.shape != q.shape or out.dtype != q.dtype:
        raise _lib.Ab2Error(-1, "q and out must be contiguous tensors of the same shape and dtype")
    check(lib.ab2_attention_decode_static(cache._h, layer, q.data_ptr(), out.data_ptr(), row0, q.shape[0],
                                          float(scale), dtype_code(q.dtype), stream_ptr()))
    return out


def attention_cached(cache, q: torch.Tensor, scale: float, layer: int = 0, row0: int = 0) -> torch.Tensor:
    """q [rows, S, n_heads, head_dim]: S new queries per sequence, causal."""
    q = _cuda(q, "q")
    out = torch.empty_like(q)
    check(lib.ab2_attention_cached(cache._h, layer, q.data_ptr(), out.data_ptr(), q.shape[1], row0, q.shape[0],
                                   float(scale), dtype_code(q.dtype), stream_ptr()))
    return out


def argmax(logits: torch.Tensor) -> torch.Tensor:
    """Greedy token per row: the last index among equal maxima."""
    logits = _cuda(logits, "logits")
    rows = logits.numel() // logits.shape[-1]
    out = torch.empty(rows, dtype=torch.int32, device=logits.device)
    check(lib.ab2_argmax(logits.data_ptr(), rows, logits.shape[-1], dtype_code(logits.dtype), out.data_ptr(),
                         stream_ptr()))
    return out


def embedding_forward(table, ids: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    ids = _cuda(ids, "ids").to(torch.int32)
    out = torch.empty((*ids.shape, table.in_features), dtype=dtype, device=ids.device)
    check(lib.ab2_embedding_forward(table._h, ids.data_ptr(), ids.numel(), out.data_ptr(), dtype_code(dtype),
                                    stream_ptr()))
    return out


# -- mechanisms of layer stacks (``model.StackConfig``), one layer of a stack cache at a time --------

def rotation_tables(positions: int, dims: int, base: float):
    """cos, sin [positions, dims / 2] (f32) of position * base ** (-2i / dims), the angles in f64."""
    f = torch.pow(torch.tensor(float(base), dtype=torch.float64), -2.0 * torch.arange(dims // 2, dtype=torch.float64) / dims)
    a = torch.arange(positions, dtype=torch.float64)[:, None] * f
    return a.cos().float().cuda(), a.sin().float().cuda()


def decay_powers(decay) -> torch.Tensor:
    """[heads, 65] f32: powers 0..64 of every head's decay."""
    d = torch.tensor(list(decay), dtype=torch.float64)[:, None]
    return torch.pow(d, torch.arange(65, dtype=torch.float64)).float().cuda().contiguous()


def window_attention(cache, cfg, layer: int, qkv: torch.Tensor, tables, eps: float, v_first=None, v_mode: int = 0,
                     row0: int = 0) -> torch.Tensor:
    """qkv [rows, S, heads dim + kv_heads dim + kv_heads vdim] (overwritten) -> [rows, S, heads vdim]."""
    qkv = _cuda(qkv, "qkv")
    specs, _keep = cfg.c_specs()
    sp = specs[layer]
    rows, S = qkv.shape[:2]
    out = torch.empty((rows, S, sp.heads * sp.vdim), dtype=qkv.dtype, device=qkv.device)
    cos, sin = tables if tables is not None else (None, None)
    check(lib.ab2_window_attention(cache._h, layer, C.byref(sp), qkv.data_ptr(), v_first.data_ptr() if v_first is not None else None,
                                   v_mode, cos.data_ptr() if cos is not None else None, sin.data_ptr() if sin is not None else None,
                                   float(eps), out.data_ptr(), S, row0, rows, dtype_code(qkv.dtype), stream_ptr()))
    return out


def lightning_scratch(cfg, layer: int) -> torch.Tensor:
    """Scratch with which a long prompt of a lightning layer runs in segments side by side."""
    m = cfg.layers[layer][0]
    return torch.empty(16 * m.heads * m.dim * m.vdim, dtype=torch.float32, device="cuda")


def lightning_attention(cache, cfg, layer: int, qkv: torch.Tensor, powers: torch.Tensor, row0: int = 0,
                        scratch: torch.Tensor | None = None) -> torch.Tensor:
    """qkv [rows, S, stride] starting with heads dim | heads dim | heads vdim -> f32 [rows, S, heads vdim]."""
    qkv = _cuda(qkv, "qkv")
    specs, _keep = cfg.c_specs()
    sp = specs[layer]
    rows, S, stride = qkv.shape
    out = torch.empty((rows, S, sp.heads * sp.vdim), dtype=torch.float32, device=qkv.device)
    check(lib.ab2_lightning_attention(cache._h, layer, C.byref(sp), powers.data_ptr(), qkv.data_ptr(), stride,
                                      scratch.data_ptr() if scratch is not None else None, out.data_ptr(), S, row0,
                                      rows, dtype_code(qkv.dtype), stream_ptr()))
    return out


def latent_attention(cache, cfg, layer: int, proj: torch.Tensor, norm: torch.Tensor, ukv, tables, eps: float, row0: int = 0,
                     workspace: torch.Tensor | None = None, reuse: bool = False) -> torch.Tensor:
    """proj [rows, S, stride] (overwritten): heads (dim + rot_dims) queries | latent | shared key part | gates;
    ``ukv`` the keys' and values' up projection (``QuantLinear``) -> [rows, S, heads vdim].  With ``reuse`` the
    workspace is that of an earlier call with the same ``ukv``."""
    proj = _cuda(proj, "proj")
    specs, _keep = cfg.c_specs(cfg.runs())
    sp = specs[layer]
    rows, S, stride = proj.shape
    if workspace is None:
        n = C.c_size_t()
        check(lib.ab2_latent_workspace(C.byref(sp), rows * S, cache.cap, dtype_code(proj.dtype), C.byref(n)))
        workspace = torch.empty(n.value, dtype=torch.uint8, device=proj.device)
    out = torch.empty((rows, S, sp.heads * sp.vdim), dtype=proj.dtype, device=proj.device)
    cos, sin = tables if tables is not None else (None, None)
    check(lib.ab2_latent_attention(cache._h, layer, C.byref(sp), proj.data_ptr(), stride, norm.data_ptr(), ukv._h,
                                   cos.data_ptr() if cos is not None else None, sin.data_ptr() if sin is not None else None, float(eps),
                                   out.data_ptr(), workspace.data_ptr(), workspace.numel(), int(reuse), S, row0, rows, dtype_code(proj.dtype), stream_ptr()))
    return out


def poly_norm(z: torch.Tensor, coef, eps: float) -> torch.Tensor:
    """a N(z) + b N(z^2) + c N(z^3) + e over the last dimension, N the division by the root mean square."""
    z = _cuda(z, "z")
    out = torch.empty_like(z)
    check(lib.ab2_poly_norm(z.data_ptr(), out.data_ptr(), z.numel() // z.shape[-1], z.shape[-1], (C.c_float * 4)(*coef), float(eps),
                            dtype_code(z.dtype), stream_ptr()))
    return out


class MoeExperts:
    """The feed-forward of a ``model.MoeFfn`` with a router over dense bf16 weights: x [tokens, width] -> the chosen
    experts' outputs [tokens, top, width] (f32; their sum is the layer's output)."""

    def __init__(self, ffn, router, gate, up, down):
        self.spec = _lib.LayerSpec(ffn=_lib.FFN_MOE, experts=ffn.experts, top=ffn.top, ff=ffn.ff, limit=ffn.limit, glu=_lib.GLU[ffn.glu])
        self.router, self.gate, self.up, self.down = router, gate, up, down
        self._work = None

    def __call__(self, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        x = _cuda(x, "x")
        T, width = x.shape
        n = C.c_size_t()
        check(lib.ab2_moe_workspace(C.byref(self.spec), width, T, dtype_code(x.dtype), C.byref(n)))
        if self._work is None or self._work.numel() < n.value:
            self._work = torch.empty(n.value, dtype=torch.uint8, device=x.device)
        if out is None:
            out = torch.empty((T, self.spec.top, width), dtype=torch.float32, device=x.device)
        check(lib.ab2_moe_forward(C.byref(self.spec), self.router._h, self.gate._h, self.up._h, self.down._h, x.data_ptr(), T,
                                  dtype_code(x.dtype), out.data_ptr(), self._work.data_ptr(), stream_ptr()))
        return out


# -- a serving step over a paged cache (``kvcache.PagedKVCache`` keeps the pages) ---------------------
# Plain calls (contiguous tensors that match) are made by csrc/fast.cpp, which answers None to all others; they are looked at here.  The same
# kernels either way: where that module does not load (it is built for one Python and one torch) a call takes some 8 us more of host time.
try:
    from . import _fast
except ImportError:
    _fast = None


@dataclass
class RotaryScaling:
    """How frequencies are changed for contexts longer than the one learnt, ``factor`` times as long.  ``linear``: every
    frequency divided by it.  ``base``: the base times factor ** (dims / (dims - 2)), so that the fastest pair stays and the slowest is
    divided by it.  ``ramp``: pairs that turn at least ``high`` times over the ``original`` context stay, those that turn at most
    ``low`` times are divided, the others lie between, linearly in their turns; magnitude 0.1 ln(factor) + 1."""
    kind: str
    factor: float
    original: int = 0
    low: float = 1.0
    high: float = 32.0

    @property
    def magnitude(self) -> float:
        return 0.1 * math.log(self.factor) + 1.0 if self.kind == "ramp" and self.factor > 1 else 1.0


def rotary_frequencies(dims: int, base: float = 10000.0, scaling: RotaryScaling | None = None, device="cuda") -> torch.Tensor:
    """[dims / 2] f64: the radians a position turns each pair by, base ** (-2i / dims), scaled."""
    if dims < 2 or dims % 2:
        raise _lib.Ab2Error(-1, f"an even number of dimensions is rotated, got {dims}")
    if not base > 0:
        raise _lib.Ab2Error(-7, f"the base of the frequencies must be positive, got {base}")
    if scaling is not None:
        if scaling.kind not in ("linear", "base", "ramp") or not scaling.factor > 0:
            raise _lib.Ab2Error(-7, f"unknown scaling {scaling}")
        if scaling.kind == "base":
            if dims == 2:
                raise _lib.Ab2Error(-1, "a single pair has no base to scale")
            base = base * scaling.factor ** (dims / (dims - 2))
    f = torch.pow(torch.tensor(float(base), dtype=torch.float64), -2.0 * torch.arange(dims // 2, dtype=torch.float64) / dims)
    if scaling is not None and scaling.kind == "linear":
        f = f / scaling.factor
    elif scaling is not None and scaling.kind == "ramp":
        if scaling.original <= 0 or not scaling.high > scaling.low:
            raise _lib.Ab2Error(-7, f"a ramp needs the original context and high > low, got {scaling}")
        turns = scaling.original * f / (2 * math.pi)
        keep = ((turns - scaling.low) / (scaling.high - scaling.low)).clamp(0, 1)
        f = f * keep + f / scaling.factor * (1 - keep)
    return f.to(device)


def _on_device(*tensors) -> None:
    """Kernels run on the current device's stream: every tensor has to be there."""
    here = None
    for t in tensors:
        if t is None:
            continue
        at = t.get_device()   # -1 for host memory
        if at != here:   # the first one, or a wrong one
            if here is not None or at < 0 or at != torch.cuda.current_device():
                raise _lib.Ab2Error(-7, f"tensors must be on the current CUDA device (this library has no CPU path), got one on {t.device}")
            here = at


def _typed(t: torch.Tensor, dtype: torch.dtype, shape: tuple, what: str) -> torch.Tensor:
    if t.dtype is not dtype:
        raise _lib.Ab2Error(-3, f"{what} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise _lib.Ab2Error(-1, f"{what} must have shape {list(shape)}, got {list(t.shape)}")
    return t if t.is_contiguous() else t.contiguous()


def _heads(t: torch.Tensor, what: str):
    """A [tokens, heads, dim] tensor whose tokens may lie apart (q of a fused projection): itself or a copy, and the elements
    from one token to the next."""
    if t.dim() != 3:
        raise _lib.Ab2Error(-1, f"{what} must be [tokens, heads, head_dim], got {list(t.shape)}")
    n, h, d = t.shape
    s0, s1, s2 = t.stride()
    if (s2 == 1 or d == 1) and (s1 == d or h == 1) and (s0 >= h * d or n < 2):
        return t, (s0 if n > 1 else h * d)
    return t.contiguous(), h * d


def _fresh(t: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor like t."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty_like(t, memory_format=torch.contiguous_format)


def _rotation(frequencies, layout: str, dim: int):
    if layout not in _lib.ROTARY:
        raise _lib.Ab2Error(-7, f"unknown rotary layout {layout!r}")
    if frequencies is None:
        return None, 0
    n = frequencies.numel()
    if 2 * n > dim:
        raise _lib.Ab2Error(-1, f"{n} pairs do not fit a head of {dim}")
    return _typed(frequencies, torch.float64, (n,), "frequencies"), 2 * n


def rotary_apply(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, frequencies: torch.Tensor, layout: str = "half",
                 magnitude: float = 1.0, out=None):
    """q [tokens, heads, dim] and k [tokens, kv_heads, dim] (or None), each token rotated by its position (``positions`` [tokens],
    int32 or int64); pairs ``half`` (i, i + n) or ``interleaved`` (2i, 2i + 1), n the count of ``frequencies`` (``rotary_frequencies``).
    ``out``: a pair of tensors for the results, which may be q and k."""
    if out is None and _fast is not None:
        got = _fast.rotary(q, k, positions, frequencies, layout, magnitude)
        if got is not None:
            return got if type(got) is tuple else check(got)
    _on_device(q, k, positions, frequencies)
    q, qs = _heads(q, "q")
    n, h, d = q.shape
    ks = kv = 0
    if k is not None:
        k, ks = _heads(k, "k")
        kv = k.shape[1]
        if k.shape[0] != n or k.shape[2] != d or k.dtype != q.dtype:
            raise _lib.Ab2Error(-1, f"q {list(q.shape)} {q.dtype} and k {list(k.shape)} {k.dtype} do not match")
    if positions.dtype not in (torch.int32, torch.int64):
        raise _lib.Ab2Error(-3, f"positions must be int32 or int64, got {positions.dtype}")
    positions = _typed(positions, positions.dtype, (n,), "positions")
    frequencies, rot = _rotation(frequencies, layout, d)
    if out is None:
        qo, qos, ko, kos = _fresh(q), h * d, None, kv * d
        if k is not None:
            ko = _fresh(k)
    else:
        qo, qos = _result(out[0], q, "out[0]")
        ko, kos = _result(out[1], k, "out[1]") if k is not None else (None, 0)
    check(lib.ab2_rotary_apply(q.data_ptr(), qs, h, k.data_ptr() if k is not None else None, ks, kv, d, positions.data_ptr(),
                               positions.dtype == torch.int64, n, frequencies.data_ptr() if frequencies is not None else None, rot, _lib.ROTARY[layout], magnitude,
                               qo.data_ptr(), qos, ko.data_ptr() if ko is not None else None, kos, dtype_code(q.dtype), stream_ptr()))
    return qo, ko


def _result(out: torch.Tensor, like: torch.Tensor, what: str):
    """A caller's tensor for a result, and its token stride; it is written in place, so no copy will do."""
    _on_device(out)
    if out.shape != like.shape or out.dtype != like.dtype:
        raise _lib.Ab2Error(-1, f"{what} must be {like.dtype} {list(like.shape)}, got {out.dtype} {list(out.shape)}")
    same, stride = _heads(out, what)
    if same is not out:
        raise _lib.Ab2Error(-1, f"{what}'s heads must lie one after the other")
    return out, stride


def _paged(k_pages, v_pages, table, lens, starts, tokens: int):
    """ab2_paged of a layer's pages and a batch, and the tensors it points to."""
    if k_pages.dim() != 4 or v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype:
        raise _lib.Ab2Error(-1, f"pages must be two tensors [pages, kv_heads, page_size, head_dim] of one type, got {list(k_pages.shape)} and {list(v_pages.shape)}")
    if not (k_pages.is_contiguous() and v_pages.is_contiguous()):
        raise _lib.Ab2Error(-1, "pages must be contiguous")
    if table.dim() != 2 or table.dtype != torch.int32:
        raise _lib.Ab2Error(-1, f"the table must be int32 [rows, pages], got {table.dtype} {list(table.shape)}")
    rows, width = table.shape
    if width > 1 and table.stride(1) != 1 or rows > 1 and table.stride(0) < width:
        table = table.contiguous()
    lens = _typed(lens, torch.int32, (rows,), "lens")
    if starts is not None:
        starts = _typed(starts, torch.int32, (rows + 1,), "starts")
    pages, kv, page, dim = k_pages.shape
    c = _lib.Paged(k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), lens.data_ptr(), starts.data_ptr() if starts is not None else None,
                   pages, page, kv, dim, width, rows, tokens, table.stride(0) if rows > 1 else width)
    return c, (table, lens, starts)


def paged_append(k_pages: torch.Tensor, v_pages: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                 starts: torch.Tensor | None = None, q: torch.Tensor | None = None, frequencies: torch.Tensor | None = None, layout: str = "half",
                 magnitude: float = 1.0, out: torch.Tensor | None = None):
    """Writes the new tokens' k (rotated at their positions in their rows, as they are without ``frequencies``) and v
    [tokens, kv_heads, dim] to the pages that ``table`` [rows, pages] names; ``lens`` [rows] are the rows' tokens with the new ones,
    ``starts`` [rows + 1] where a row's new tokens begin (None: one a row).  Returns the rotated q [tokens, heads, dim], if any."""
    if out is None and _fast is not None:
        got = _fast.append(k_pages, v_pages, k, v, table, lens, starts, q, frequencies, layout, magnitude)
        if got is not None:
            return check(got) if type(got) is int else got if got is not True else None
    _on_device(k_pages, v_pages, k, v, table, lens, starts, q, frequencies)
    k, ks = _heads(k, "k")
    v, vs = _heads(v, "v")
    n, kv, d = k.shape
    if v.shape != k.shape or v.dtype != k.dtype or k.dtype != k_pages.dtype:
        raise _lib.Ab2Error(-1, f"k {list(k.shape)} {k.dtype} and v {list(v.shape)} {v.dtype} do not match each other and pages of {k_pages.dtype}")
    c, _keep = _paged(k_pages, v_pages, table, lens, starts, n)
    if (kv, d) != (c.kv_heads, c.head_dim):
        raise _lib.Ab2Error(-1, f"k has {kv} heads of {d}, the pages {c.kv_heads} of {c.head_dim}")
    frequencies, rot = _rotation(frequencies, layout, d)
    h = qs = qos = 0
    qo = None
    if q is not None:
        q, qs = _heads(q, "q")
        h = q.shape[1]
        if q.shape[0] != n or q.shape[2] != d or q.dtype != k.dtype:
            raise _lib.Ab2Error(-1, f"q {list(q.shape)} {q.dtype} does not match k {list(k.shape)} {k.dtype}")
        if out is None:
            qo, qos = _fresh(q), h * d
        else:
            qo, qos = _result(out, q, "out")
    check(lib.ab2_paged_append(C.byref(c), k.data_ptr(), ks, v.data_ptr(), vs, q.data_ptr() if q is not None else None, qs, h,
                               qo.data_ptr() if qo is not None else None, qos, frequencies.data_ptr() if frequencies is not None else None, rot,
                               _lib.ROTARY[layout], magnitude, dtype_code(k.dtype), stream_ptr()))
    return qo


def attention_paged(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, scale: float,
                    starts: torch.Tensor | None = None, max_new: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """q [tokens, heads, dim]: each row's new tokens, whose keys and values have been appended, attend to the row's keys up to their
    own; table, lens and starts as in ``paged_append``.  ``max_new`` bounds the new tokens of a row (None: not known); it picks
    kernels, whose results differ by rounding.  Over bf16 a softmax weight keeps 16 bits where a row's new tokens times the query heads of a KV head are
    at most 16, and 8 where they are more.  Tokens behind the last row are left as ``out`` (not q) holds them."""
    if out is None and _fast is not None:
        got = _fast.attention(q, k_pages, v_pages, table, lens, scale, starts, max_new)
        if got is not None:
            return check(got) if type(got) is int else got
    _on_device(q, k_pages, v_pages, table, lens, starts)
    q, qs = _heads(q, "q")
    n, h, d = q.shape
    if q.dtype != k_pages.dtype:
        raise _lib.Ab2Error(-3, f"queries of {q.dtype} over pages of {k_pages.dtype}")
    c, _keep = _paged(k_pages, v_pages, table, lens, starts, n)
    if d != c.head_dim:
        raise _lib.Ab2Error(-1, f"queries have heads of {d}, the pages of {c.head_dim}")
    if (q.data_ptr() | qs * q.element_size()) & 15:
        q, qs = q.clone(memory_format=torch.contiguous_format), h * d
    if out is None:
        out, os = _fresh(q), h * d
    else:
        out, os = _result(out, q, "out")
    max_new = (1 if starts is None else max(n, 1)) if max_new is None else min(max_new, 2 ** 31 - 1)
    size = C.c_size_t()
    if c.table_width * c.page_size > _lib.PAGED_UNCUT:
        check(lib.ab2_paged_workspace(d, C.byref(size)))
    size = size.value
    work = torch.empty(size, dtype=torch.uint8, device=q.device) if size else None
    check(lib.ab2_paged_attention(C.byref(c), q.data_ptr(), qs, h, out.data_ptr(), os, max_new, scale, work.data_ptr() if size else None, size,
                                  dtype_code(q.dtype), stream_ptr()))
    return out


def allowed_words(mask: torch.Tensor) -> torch.Tensor:
    """A truth value for every token [rows, vocab] as the words that ``adjust_logits`` takes: int32 [rows, ceil(vocab / 32)]."""
    if mask.dim() != 2:
        raise _lib.Ab2Error(-1, f"a mask must be [rows, vocab], got {list(mask.shape)}")
    rows, vocab = mask.shape
    bits = torch.zeros((rows, (vocab + 31) // 32 * 32), dtype=torch.int64, device=mask.device)
    bits[:, :vocab] = mask != 0
    words = (bits.view(rows, -1, 32) << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32)


def adjust_logits(logits: torch.Tensor, history: torch.Tensor | None = None, lengths: torch.Tensor | None = None, rules: torch.Tensor | None = None,
                  bias_ids: torch.Tensor | None = None, bias_values: torch.Tensor | None = None, allowed: torch.Tensor | None = None,
                  out: torch.Tensor | None = None) -> torch.Tensor:
    """The rules of a sampler on logits [rows, vocab]; ``argmax`` picks from the result.

    With c the times a token occurs in ``history`` [rows, n] int32 (the first ``lengths`` [rows] of a row, None: all; ids outside the
    vocabulary are passed over) and ``rules`` [rows, 3] f32 = (repetition > 0, presence, frequency): a token with c > 0 has its logit divided
    by the repetition where it is positive, else multiplied, then lowered by presence + frequency c.  Then ``bias_values`` [rows, m] f32 are
    added at ``bias_ids`` [rows, m] int32 (of an id named twice the last counts), and tokens whose bit in ``allowed``
    [rows, ceil(vocab / 32)] int32 (``allowed_words``) is 0 become -inf.  ``out`` may be the logits."""
    if out is None and _fast is not None:
        got = _fast.logits(logits, history, lengths, rules, bias_ids, bias_values, allowed)
        if got is not None:
            return check(got) if type(got) is int else got
    _on_device(logits, history, lengths, rules, bias_ids, bias_values, allowed, out)
    if logits.dim() != 2:
        raise _lib.Ab2Error(-1, f"logits must be [rows, vocab], got {list(logits.shape)}")
    rows, vocab = logits.shape
    if vocab > 1 and logits.stride(1) != 1 or rows > 1 and logits.stride(0) < vocab:
        logits = logits.contiguous()
    stride = logits.stride(0) if rows > 1 else vocab
    hp = lp = rp = bp = vp = ap = None
    hs = width = biases = 0
    if history is not None:
        if rules is None:
            raise _lib.Ab2Error(-7, "a history needs rules")
        if history.dim() != 2 or history.shape[0] != rows or history.dtype != torch.int32:
            raise _lib.Ab2Error(-1, f"history must be int32 [{rows}, tokens], got {history.dtype} {list(history.shape)}")
        width = history.shape[1]
        if width > 1 and history.stride(1) != 1 or rows > 1 and history.stride(0) < width:
            history = history.contiguous()
        hp, hs = history.data_ptr(), (history.stride(0) if rows > 1 else width)
        rules = _typed(rules, torch.float32, (rows, 3), "rules")
        rp = rules.data_ptr()
        if lengths is not None:
            lengths = _typed(lengths, torch.int32, (rows,), "lengths")
            lp = lengths.data_ptr()
    elif lengths is not None or rules is not None:
        raise _lib.Ab2Error(-7, "lengths and rules are those of a history")
    if (bias_ids is None) != (bias_values is None):
        raise _lib.Ab2Error(-7, "biases need both ids and values")
    if bias_ids is not None:
        biases = bias_ids.shape[-1]
        bias_ids = _typed(bias_ids, torch.int32, (rows, biases), "bias_ids")
        bias_values = _typed(bias_values, torch.float32, (rows, biases), "bias_values")
        bp, vp = bias_ids.data_ptr(), bias_values.data_ptr()
    if allowed is not None:
        allowed = _typed(allowed, torch.int32, (rows, (vocab + 31) // 32), "allowed")
        ap = allowed.data_ptr()
    if out is None:
        out = _fresh(logits)
    elif out.shape != logits.shape or out.dtype != logits.dtype or not out.is_contiguous():
        raise _lib.Ab2Error(-1, f"out must be contiguous {logits.dtype} {list(logits.shape)}")
    check(lib.ab2_adjust_logits(logits.data_ptr(), stride, rows, vocab, hp, hs, width, lp, rp, bp, vp, biases, ap, out.data_ptr(),
                                dtype_code(logits.dtype), stream_ptr()))
    return out
