"""Host-side mirror of the reference's KV caches.

``KVCache`` follows ``KVCache`` of crates/aarambh-studio-nn/src/kvcache.rs:236-369
(update / truncate / clear / seq_len / capacity) for ``batch`` independent
sequences, and with ``n_layers > 1`` the engine-level ``KvCache`` of
crates/aarambh-studio-inference/src/kvcache.rs:7-80 (one length shared by all
layers, snapshot / restore).  Storage is f32, bf16 or per-token-per-head INT8.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass, field

import torch

from . import _lib
from ._lib import check, lib
from .qlinear import dtype_code, stream_ptr

_KV_DTYPES = {"f32": _lib.KV_F32, "bf16": _lib.KV_BF16, "int8": _lib.KV_INT8}


class KVCache:
    def __init__(self, capacity: int, kv_heads: int, head_dim: int, n_heads: int, batch: int = 1,
                 n_layers: int = 1, dtype: str = "f32", _handle=None):
        self.cap, self.kv_heads, self.head_dim, self.n_heads = capacity, kv_heads, head_dim, n_heads
        self.batch, self.n_layers, self.dtype = batch, n_layers, dtype
        if _handle is None:
            h = C.c_void_p()
            check(lib.ab2_kv_create(C.byref(h), n_layers, batch, capacity, kv_heads, head_dim, n_heads,
                                    _KV_DTYPES[dtype]))
            _handle = h.value
        self._h = C.c_void_p(_handle)

    @classmethod
    def with_capacity(cls, capacity, kv_heads, head_dim, n_heads, **kw):
        return cls(capacity, kv_heads, head_dim, n_heads, **kw)

    @classmethod
    def for_stack(cls, cfg, capacity: int, batch: int, max_step: int, dtype: str):
        """The cache of a layer stack (``StackConfig``): windows in rings, latents, recurrent states beside them;
        one cache layer for every run of a layer."""
        order = cfg.runs()
        specs, _keep = cfg.c_specs(order)
        h = C.c_void_p()
        check(lib.ab2_kv_create_stack(C.byref(h), specs, len(order), batch, capacity, max_step, _KV_DTYPES[dtype]))
        return cls(capacity, 0, 0, 0, batch, len(order), dtype, _handle=h.value)

    def update(self, k: torch.Tensor, v: torch.Tensor, row0: int = 0):
        """Appends k, v [rows, S, kv_heads, head_dim] and returns the cached tensors
        of the first row touched, dequantised ([len, kv_heads, head_dim])."""
        if k.dim() != 4 or v.shape != k.shape:
            raise _lib.Ab2Error(-1, f"KV cache expects matching rank-4 tensors, got {tuple(k.shape)} and {tuple(v.shape)}")
        k = k.contiguous(); v = v.contiguous()
        check(lib.ab2_kv_update(self._h, k.data_ptr(), v.data_ptr(), k.shape[1], row0, k.shape[0],
                                dtype_code(k.dtype), stream_ptr()))
        return self.read(row0)

    def append(self, layer, k, v, row0=0, cos=None, sin=None, positions=None, max_seq=0):
        k = k.contiguous(); v = v.contiguous()
        check(lib.ab2_kv_append(self._h, layer, k.data_ptr(), v.data_ptr(), k.shape[1], row0, k.shape[0],
                                dtype_code(k.dtype), cos.data_ptr() if cos is not None else None,
                                sin.data_ptr() if sin is not None else None,
                                positions.data_ptr() if positions is not None else None, max_seq,
                                stream_ptr()))

    def commit(self, S, row0=0, nrows=None):
        check(lib.ab2_kv_commit(self._h, S, row0, self.batch - row0 if nrows is None else nrows, stream_ptr()))

    def read(self, row: int = 0, layer: int = 0):
        n = self.seq_len(row)
        k = torch.empty((n, self.kv_heads, self.head_dim), dtype=torch.float32, device="cuda")
        v = torch.empty_like(k)
        check(lib.ab2_kv_read(self._h, layer, row, k.data_ptr(), v.data_ptr(), stream_ptr()))
        return k, v

    def truncate(self, new_len: int, row: int = 0):
        check(lib.ab2_kv_truncate(self._h, row, new_len, stream_ptr()))

    def save_row(self, row: int = 0):
        """Remembers a row's recurrent states, so that ``truncate`` to its present length can restore them."""
        check(lib.ab2_kv_save_row(self._h, row, stream_ptr()))

    def has_state(self) -> bool:
        """Whether a layer keeps a recurrent state (its rows are cut to 0 or to a saved length only)."""
        n = C.c_int()
        check(lib.ab2_kv_has_state(self._h, C.byref(n)))
        return bool(n.value)

    def clear(self):
        check(lib.ab2_kv_clear(self._h, stream_ptr()))

    def seq_len(self, row: int = 0) -> int:
        n = C.c_int()
        check(lib.ab2_kv_seq_len(self._h, row, C.byref(n)))
        return n.value

    def capacity(self) -> int:
        n = C.c_int()
        check(lib.ab2_kv_capacity(self._h, C.byref(n)))
        return n.value

    def snapshot(self) -> "KVCache":
        h = C.c_void_p()
        check(lib.ab2_kv_clone(C.byref(h), self._h, stream_ptr()))
        return KVCache(self.cap, self.kv_heads, self.head_dim, self.n_heads, self.batch, self.n_layers,
                       self.dtype, _handle=h.value)

    def restore(self, snapshot: "KVCache"):
        """Takes over the snapshot's storage (KvCache::restore)."""
        old = self._h
        self._h, snapshot._h = snapshot._h, None
        lib.ab2_kv_destroy(old)

    def __del__(self):
        try:
            if self._h:
                lib.ab2_kv_destroy(self._h)
                self._h = None
        except Exception:
            pass


@dataclass
class PagedStep:
    """The new tokens of some rows of a paged cache, on the device: what ``paged_append`` and ``attention_paged`` read."""
    rows: list
    new: list                     # new tokens of each
    table: torch.Tensor           # [rows, pages]
    lens: torch.Tensor            # [rows], new tokens included
    starts: torch.Tensor          # [rows + 1]
    tokens: int                   # that q, k and v have room for
    max_new: int
    packed: torch.Tensor          # the three above
    before: list = field(default_factory=list)   # tokens of each row without the new ones (empty in a step that a caller put together: it is not looked at)
    cuts: list = field(default_factory=list)     # how often each row had been cut back, and all rows together
    all_cuts: int = 0


class PagedKVCache:
    """Keys and values in pages of one pool that the sequences share: a sequence holds as many as its tokens need, in any order, where
    ``KVCache`` gives each the same capacity for good.  ``k`` and ``v`` are [layers, pages, kv_heads, page_size, head_dim] (f32, bf16, or e4m3 with
    ``k_scales`` and ``v_scales`` [layers, pages, kv_heads, page_size / 16] f32: half the room of bf16, for queries, keys and values of bf16 or f32).
    A pass over some rows: ``step`` takes the pages it needs, then for every layer ``append`` and ``attention``, at its end ``commit``.  A step whose rows
    have been cut back or have moved on since is refused: its pages may be another row's.
    Calls on a cache go on one stream, or are ordered by the caller."""

    def __init__(self, pages: int, page_size: int, kv_heads: int, head_dim: int, batch: int = 1, n_layers: int = 1, dtype: str = "bf16", device="cuda"):
        if dtype not in ("f32", "bf16", "e4m3"):
            raise _lib.Ab2Error(-3, f"paged caches hold f32, bf16 or e4m3, not {dtype}")
        if page_size not in (16, 32, 64, 128, 256) or head_dim not in (64, 128):
            raise _lib.Ab2Error(-8, f"pages of {page_size} tokens, heads of {head_dim}: 16, 32, 64, 128 or 256 tokens and heads of 64 or 128 are served")
        if min(pages, kv_heads, batch, n_layers) <= 0:
            raise _lib.Ab2Error(-1, f"paged cache of {pages} pages, {kv_heads} heads, {batch} rows, {n_layers} layers")
        self.page_size, self.kv_heads, self.head_dim, self.batch, self.n_layers, self.dtype = page_size, kv_heads, head_dim, batch, n_layers, dtype
        kind = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}[dtype]
        self.k, self.v = (torch.zeros((n_layers, pages, kv_heads, page_size, head_dim), dtype=kind, device=device) for _ in range(2))
        self.k_scales = self.v_scales = None
        if dtype == "e4m3":
            self.k_scales, self.v_scales = (torch.zeros((n_layers, pages, kv_heads, page_size // _lib.PAGED_BLOCK), dtype=torch.float32, device=device) for _ in range(2))
        self._free = list(range(pages - 1, -1, -1))
        self._pages = [[] for _ in range(batch)]
        self._lens = [0] * batch
        self._cuts, self._all_cuts = [0] * batch, 0

    def _row(self, row: int) -> int:
        if not 0 <= row < self.batch:
            raise _lib.Ab2Error(-7, f"row {row} of a cache of {self.batch}")
        return row

    def free_pages(self) -> int:
        return len(self._free)

    def seq_len(self, row: int = 0) -> int:
        return self._lens[self._row(row)]

    def reserve(self, row: int, tokens: int) -> None:
        """Takes the pages that ``tokens`` more tokens of a row need (AB2_ERR_CAPACITY, and none taken, where they are not to be had)."""
        need = -(-(self.seq_len(row) + tokens) // self.page_size) - len(self._pages[row])
        if need > len(self._free):
            raise _lib.Ab2Error(-4, f"row {row} needs {need} more pages, {len(self._free)} are free")
        for _ in range(need):
            self._pages[row].append(self._free.pop())

    def step(self, rows, new, room: int = 0, into: PagedStep | None = None) -> PagedStep:
        """The batch of ``new[i]`` new tokens (0 or more) of row ``rows[i]``, with pages for them.  ``room``: the table is wide enough for that many
        more tokens of each row.  ``into``: an earlier step over as many rows is written anew in place, for passes that were recorded with it."""
        rows, new = [int(r) for r in rows], [int(n) for n in new]
        if not rows or len(rows) != len(new) or min(new) < 0 or len(set(rows)) != len(rows):
            raise _lib.Ab2Error(-1, f"a step takes distinct rows and new tokens of each, got rows {rows}, new {new}")
        if room < 0:
            raise _lib.Ab2Error(-1, f"room for {room} more tokens")
        for r in rows:
            self._row(r)
        lens = [self._lens[r] + n for r, n in zip(rows, new)]
        short = sum(max(0, -(-l // self.page_size) - len(self._pages[r])) for r, l in zip(rows, lens))
        if short > len(self._free):
            raise _lib.Ab2Error(-4, f"the step needs {short} more pages, {len(self._free)} are free")
        widest = max(1, max(max(len(self._pages[r]), -(-(l + room) // self.page_size)) for r, l in zip(rows, lens)))
        n, total, most = len(rows), sum(new), max(max(new), 1)
        if into is None:
            width = 1 << (widest - 1).bit_length()
            packed = torch.empty(2 * n + 1 + n * width, dtype=torch.int32, device=self.k.device)
            into = PagedStep(rows, new, packed[2 * n + 1:].view(n, width), packed[n + 1:2 * n + 1], packed[:n + 1], total, most, packed)
        elif into.table.shape[0] != n or into.table.shape[1] < widest or into.tokens < total or into.max_new < most:
            raise _lib.Ab2Error(-1, f"the step has {into.table.shape[0]} rows of {into.table.shape[1]} pages, {into.tokens} tokens, {into.max_new} a row: "
                                    f"{n} rows of {widest}, {total}, {most} do not fit")
        for r, c in zip(rows, new):
            self.reserve(r, c)
        width = into.table.shape[1]
        flat = [0]
        for c in new:
            flat.append(flat[-1] + c)
        flat += lens
        for r in rows:
            flat += self._pages[r] + [0] * (width - len(self._pages[r]))
        into.packed.copy_(torch.tensor(flat, dtype=torch.int32))
        into.rows, into.new = rows, new
        into.before, into.cuts, into.all_cuts = [self._lens[r] for r in rows], [self._cuts[r] for r in rows], self._all_cuts
        return into

    def append(self, step: PagedStep, k: torch.Tensor, v: torch.Tensor, layer: int = 0, q: torch.Tensor | None = None, frequencies=None, layout: str = "half",
               magnitude: float = 1.0, out: torch.Tensor | None = None):
        """``dispatch.paged_append`` on a layer: k, v (and q) [step.tokens, heads, dim]."""
        from .dispatch import paged_append
        self._holds(step, k)
        return paged_append(self.k[layer], self.v[layer], k, v, step.table, step.lens, step.starts, q, frequencies, layout, magnitude, out, self._scales(layer))

    def attention(self, step: PagedStep, q: torch.Tensor, scale: float, layer: int = 0, out: torch.Tensor | None = None, window: int = 0, sinks: int = 0) -> torch.Tensor:
        """``dispatch.attention_paged`` on a layer: q [step.tokens, heads, dim]; with a ``window`` a token sees its last so many keys and the first ``sinks``."""
        from .dispatch import attention_paged
        self._holds(step, q)
        return attention_paged(q, self.k[layer], self.v[layer], step.table, step.lens, scale, step.starts, step.max_new, out, self._scales(layer), window, sinks)

    def _scales(self, layer: int):
        return None if self.k_scales is None else (self.k_scales[layer], self.v_scales[layer])

    def _holds(self, step, t=None):
        if t is not None and t.shape[0] < step.tokens:
            raise _lib.Ab2Error(-1, f"a step of {step.tokens} tokens over a tensor of {t.shape[0]}")
        if step.all_cuts != self._all_cuts and step.cuts and step.cuts != [self._cuts[r] for r in step.rows]:
            raise _lib.Ab2Error(-7, f"rows {[r for r, c in zip(step.rows, step.cuts) if c != self._cuts[r]]} were cut back behind the step's making: it needs to be made anew")

    def commit(self, step: PagedStep) -> None:
        """The rows' lengths move on by the step's new tokens, once."""
        self._holds(step)
        if step.before and step.before != [self._lens[r] for r in step.rows]:
            raise _lib.Ab2Error(-7, f"rows {[r for r, n in zip(step.rows, step.before) if n != self._lens[r]]} have moved on since the step was made")
        for r, n in zip(step.rows, step.new):
            self._lens[r] += n

    def truncate(self, new_len: int, row: int = 0) -> None:
        """Cuts a row back; pages behind its end are free again."""
        if not 0 <= new_len <= self.seq_len(row):
            raise _lib.Ab2Error(-4, f"row {row} holds {self.seq_len(row)} tokens and cannot be cut to {new_len}")
        self._lens[row] = new_len
        self._cuts[row] += 1
        self._all_cuts += 1
        keep = -(-new_len // self.page_size)
        self._free += self._pages[row][:keep - 1 if keep else None:-1]
        del self._pages[row][keep:]

    def clear(self) -> None:
        for row in range(self.batch):
            self.truncate(0, row)

    def read(self, row: int = 0, layer: int = 0):
        """The row's keys and values [len, kv_heads, head_dim] in f32."""
        n = self.seq_len(row)
        at = torch.tensor(self._pages[row], dtype=torch.int64, device=self.k.device)
        both = []
        for p, scales in ((self.k, self.k_scales), (self.v, self.v_scales)):
            if scales is None:
                x = p[layer][at]
            else:
                x = p[layer].view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * scales[layer][at].repeat_interleave(_lib.PAGED_BLOCK, dim=-1)[..., None]
            both.append(x.transpose(1, 2).reshape(-1, self.kv_heads, self.head_dim)[:n].float())
        return tuple(both)
