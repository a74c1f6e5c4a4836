"""An 8-bit cache of keys and values with one power-of-two scale for each block of 32 tokens and head, and what works on it.

``BlockCache`` is one layer's cache of any number of sequences (slots).  It needs no calibration: a block's scale follows from the rows
that are in it (include/moondream_hip.h, md_kv8_cache).  A decode step of a layer is::

    cache.append(k, v, row0=length, weights=w)          # the new tokens' rows, without weight so far
    o = cache.attention(q, length + 1, weights=w)       # ... and what they see; w: the weight that every cached row got so far
    kept, length = cache.evict(w, length + 1, keep=4096, recent=256)   # now and then: the rows of least weight leave

Everything runs on the current stream of the cache's device, allocates through torch only, never synchronises and can be captured into a
graph.  Lengths, rows and slots are int32 tensors on the device, one number per sequence; what they hold is not looked at on the host.
Like torch's operators on tensors of another stream, a call does not wait for work that other streams have queued.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Optional, Tuple

import torch

from . import _lib

BLOCK = _lib.MD_KV8_BLOCK
_BF16, _F32, _I32, _U8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8
_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def _launch(index: int, what: str, call, *args) -> None:
    """An entry point on the current stream of device ``index``, which is made the current one if it is not."""
    if _device() == index:  # (there are tensors on a device: torch has been set up)
        status = call(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = call(*args, _raw_stream(index))
    if status:
        _lib.check(status, what)


def _need(t: torch.Tensor, name: str, dtype: torch.dtype, index: int, shape: tuple) -> int:
    """The address of a contiguous tensor that is what it has to be."""
    if t.dtype is not dtype or t.shape != shape or t.get_device() != index or not t.is_contiguous():
        raise ValueError(f"{name}: {tuple(t.shape)} {t.dtype} on {t.device}, wanted contiguous {shape} {dtype} on cuda:{index}")
    return t.data_ptr()


class BlockCache:
    """``slots`` sequences of up to ``ctx`` rows (a multiple of 32 or rounded up to one), ``kv_heads`` heads of ``head_dim`` 64 or 128."""

    def __init__(self, slots: int, ctx: int, kv_heads: int, head_dim: int, device="cuda"):
        ctx = (ctx + BLOCK - 1) // BLOCK * BLOCK
        shape = (slots, kv_heads, ctx, head_dim)
        if min(shape) <= 0:
            raise ValueError(f"a cache of shape {shape}")
        k, v = (torch.zeros(shape, dtype=_U8, device=device) for _ in range(2))
        k_exp, v_exp = (torch.full((slots, kv_heads, ctx // BLOCK), 127 + _lib.MD_KV8_MIN_EXP, dtype=_U8, device=device) for _ in range(2))  # a block of zeros'
        self._take(k, v, k_exp, v_exp)

    @classmethod
    def of(cls, k: torch.Tensor, v: torch.Tensor, k_exp: torch.Tensor, v_exp: torch.Tensor) -> "BlockCache":
        """Over tensors that are there already: codes uint8 [slots, kv_heads, ctx, head_dim], scales uint8 [slots, kv_heads, ctx / 32]; slots may lie
        apart (a layer's part of all layers' slabs)."""
        cache = cls.__new__(cls)
        cache._take(k, v, k_exp, v_exp)
        return cache

    def _take(self, k, v, k_exp, v_exp) -> None:
        if k.dim() != 4 or k.shape != v.shape or k.shape[2] % BLOCK or k.shape[3] not in (64, 128):
            raise ValueError(f"keys {tuple(k.shape)} and values {tuple(v.shape)}: wanted [slots, kv_heads, ctx, 64 or 128] of one shape, ctx a multiple of {BLOCK}")
        slots, heads, ctx, dim = k.shape
        if min(k.shape) <= 0 or any(e.shape != (slots, heads, ctx // BLOCK) for e in (k_exp, v_exp)):
            raise ValueError(f"scales {tuple(k_exp.shape)}, {tuple(v_exp.shape)} for codes {tuple(k.shape)}")
        if any(t.dtype != _U8 or t.device != k.device for t in (k, v, k_exp, v_exp)):
            raise ValueError("codes and scales are uint8 tensors of one device")
        for t in (k, v, k_exp, v_exp):
            if not t[0].is_contiguous():
                raise ValueError("a slot's codes and scales have to be contiguous")
        if slots > 1 and (k.stride(0) != v.stride(0) or k_exp.stride(0) != v_exp.stride(0)):
            raise ValueError("keys and values lie in slots of different strides")
        if k.device.type != "cuda":
            raise _lib.MoondreamHipError("BlockCache needs a GPU device; there is no CPU path")
        self.k, self.v, self.k_exp, self.v_exp = k, v, k_exp, v_exp
        self.slots, self.kv_heads, self.ctx, self.head_dim = slots, heads, ctx, dim
        self.device = torch.device("cuda", k.device.index if k.device.index is not None else torch.cuda.current_device())
        self._index = self.device.index
        self._weight_shape = (slots, heads, ctx)
        self._lib = _lib.load()
        self._workspaces: dict = {}  # bytes that calls of a shape need
        stride = (k.stride(0), k_exp.stride(0)) if slots > 1 else (heads * ctx * dim, heads * ctx // BLOCK)
        self._struct = _lib.MdKv8Cache(k.data_ptr(), v.data_ptr(), k_exp.data_ptr(), v_exp.data_ptr(), stride[0], stride[1], slots, ctx, heads, dim)
        self._ref = C.byref(self._struct)

    def _per_sequence(self, t: Optional[torch.Tensor], name: str, batch: int) -> Optional[int]:
        return None if t is None else _need(t, name, _I32, self._index, (batch,))

    def _batch(self, batch: int, slot: Optional[torch.Tensor]) -> None:
        if batch <= 0 or (slot is None and batch > self.slots):
            raise ValueError(f"a batch of {batch} sequences in {self.slots} slots")

    def _rows_of(self, t: torch.Tensor, name: str) -> tuple:
        """The strides of bf16 rows [batch, tokens, heads, head_dim] that are as the kernels take them."""
        s = t.stride()
        if len(s) != 4 or t.dtype is not _BF16 or t.get_device() != self._index or t.shape[3] != self.head_dim:
            raise ValueError(f"{name}: {tuple(t.shape)} {t.dtype} on {t.device}, wanted [batch, tokens, heads, {self.head_dim}] bfloat16 on {self.device}")
        if s[3] != 1 or (s[0] | s[1] | s[2]) % 8 or t.data_ptr() % 16:
            raise ValueError(f"{name}: rows of head_dim have to be contiguous and 16-byte aligned (strides {s})")
        return s

    def append(self, k: torch.Tensor, v: torch.Tensor, row0: torch.Tensor, new: Optional[torch.Tensor] = None, slot: Optional[torch.Tensor] = None,
               weights: Optional[torch.Tensor] = None) -> None:
        """Rows row0[b] .. of every sequence from bf16 ``k``, ``v`` [batch, tokens, kv_heads, head_dim] (views of a projection's rows will do; keys
        rotated already); ``new``: how many of the tokens count, per sequence.  Rows past ``ctx`` are dropped.  The new rows are the sequence's last (what lay behind
        them in their last block is gone).  ``weights`` (fp32 [slots, kv_heads, ctx], what ``attention`` adds to): the new rows' become 0; without it they keep what an evicted
        row, or the slot's sequence before, left there.  A slot at most once."""
        ks, vs = self._rows_of(k, "k"), self._rows_of(v, "v")
        shape = k.shape
        batch, tokens, heads, _ = shape
        if v.shape != shape or heads != self.kv_heads:
            raise ValueError(f"keys {tuple(shape)} and values {tuple(v.shape)}, wanted [batch, tokens, {self.kv_heads}, {self.head_dim}]")
        self._batch(batch, slot)
        if tokens == 0:
            return
        of = (batch,)
        _launch(self._index, "md_kv8_append", self._lib.md_kv8_append_weighted, self._ref, k.data_ptr(), ks[0], ks[1], ks[2], v.data_ptr(), vs[0], vs[1], vs[2],
                None if slot is None else _need(slot, "slot", _I32, self._index, of), _need(row0, "row0", _I32, self._index, of),
                None if new is None else _need(new, "new", _I32, self._index, of), self._weights(weights, "weights"), batch, tokens)

    def read(self, row0: Optional[torch.Tensor], rows: int, kv_len: Optional[torch.Tensor] = None, slot: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Rows row0[b] .. row0[b] + rows - 1 (None: from 0) as bf16 [batch, kv_heads, rows, head_dim] keys and values, exactly what the codes stand
        for; zeros for rows outside [0, kv_len[b])."""
        given = next((t for t in (row0, kv_len, slot) if t is not None), None)
        batch = self.slots if given is None else given.numel()
        self._batch(batch, slot)
        if rows < 0:
            raise ValueError(f"{rows} rows")
        k, v = torch.empty((2, batch, self.kv_heads, rows, self.head_dim), dtype=_BF16, device=self.device).unbind(0)
        if rows:
            _launch(self._index, "md_kv8_read", self._lib.md_kv8_read, self._ref, self._per_sequence(slot, "slot", batch), self._per_sequence(row0, "row0", batch),
                    self._per_sequence(kv_len, "kv_len", batch), batch, rows, k.data_ptr(), v.data_ptr())
        return k, v

    def _weights(self, w: Optional[torch.Tensor], name: str) -> Optional[int]:
        return None if w is None else _need(w, name, _F32, self._index, self._weight_shape)

    def attention(self, q: torch.Tensor, kv_len: torch.Tensor, q_pos0: Optional[torch.Tensor] = None, q_rows: Optional[torch.Tensor] = None,
                  slot: Optional[torch.Tensor] = None, prefix_len: int = 0, scale: Optional[float] = None, max_len: Optional[int] = None,
                  weights: Optional[torch.Tensor] = None, decay: float = 1.0, out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Softmax attention of ``q`` [batch, tokens, heads, head_dim] (bf16) over the first ``kv_len[b]`` rows; returns the same shape.

        A sequence's queries are its last rows unless ``q_pos0`` says where the first one stands; each sees the rows up to its own, those in the first
        ``prefix_len`` rows all of these.  ``out`` may be ``q`` itself where no weights are wanted, and shares nothing with it otherwise.  ``q_rows``: how many of the queries count (the others' outputs stay as ``out`` has them; without
        ``out`` they are zeros).  ``max_len``: no sequence is longer (sizes the launch; longer ones are cut).  ``scale``: 1 / sqrt(head_dim).
        ``weights`` (fp32 [slots, kv_heads, ctx]) <- decay * weights + the softmax weight that every row got in this call."""
        qs = self._rows_of(q, "q")
        batch, tokens, heads, dim = q.shape
        if heads == 0 or heads % self.kv_heads:
            raise ValueError(f"{heads} query heads over {self.kv_heads} key heads")
        self._batch(batch, slot)
        if max_len is not None and max_len <= 0 or prefix_len < 0:
            raise ValueError(f"max_len {max_len}, prefix_len {prefix_len}")
        if out is None:
            out = (torch.empty if q_rows is None else torch.zeros)(q.shape, dtype=_BF16, device=self.device)
            os = out.stride()
        else:
            if out.shape != q.shape:
                raise ValueError(f"out: {tuple(out.shape)}, wanted {tuple(q.shape)}")
            os = self._rows_of(out, "out")
            if any(s == 0 and n > 1 for s, n in zip(os, q.shape)):  # (an expanded dimension: outputs would be written over one another)
                raise ValueError(f"out: strides {os}")
        if tokens == 0:
            return out
        longest = 0 if max_len is None else min(max_len, self.ctx)
        a = _lib.MdKv8AttnArgs(q.data_ptr(), qs[0], qs[1], qs[2], out.data_ptr(), os[0], os[1], os[2], batch, heads, tokens,
                               self._per_sequence(slot, "slot", batch), self._per_sequence(q_pos0, "q_pos0", batch),
                               self._per_sequence(q_rows, "q_rows", batch), _need(kv_len, "kv_len", _I32, self._index, (batch,)), longest,
                               min(prefix_len, self.ctx), 1.0 / math.sqrt(dim) if scale is None else scale, decay, self._weights(weights, "weights"), None, 0)
        shape = (batch, heads, tokens, longest, weights is None)
        need = self._workspaces.get(shape)
        if need is None:
            if len(self._workspaces) >= 1024:  # (max_len may be another in every step)
                self._workspaces.clear()
            need = self._workspaces[shape] = self._lib.md_kv8_attention_workspace_bytes(self._ref, C.byref(a))
        if need:
            ws = torch.empty(need, dtype=_U8, device=self.device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        _launch(self._index, "md_kv8_attention", self._lib.md_kv8_attention, self._ref, C.byref(a))
        return out

    def evict(self, weights: torch.Tensor, kv_len: torch.Tensor, keep: int, first: int = 0, recent: int = 0, slot: Optional[torch.Tensor] = None,
              into: Optional["BlockCache"] = None, into_weights: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """Of every sequence and head ``keep`` rows stay: the ``first`` ones, the ``recent`` last ones, and those of the largest ``weights`` (fp32
        [slots, kv_heads, ctx]; ties: the lower row).  They move together, in their order, to the rows 0 .. of the same slot -- of this
        cache, or of ``into``, another of as many heads that shares no memory with it -- and their weights with them (in place, or to ``into_weights``
        [slots, kv_heads, ctx] of ``into``); what lies behind the last that stayed is left as it is (``append`` clears the weights of rows that come there).  Returns the rows that stayed, int32 [batch, kv_heads, keep], -1 behind the last, and the new lengths."""
        to = self if into is None else into
        if to.device != self.device or (to.kv_heads, to.head_dim) != (self.kv_heads, self.head_dim):
            raise ValueError("into: a cache of as many heads of the same size on the same device")
        if into is None and into_weights is not None:
            raise ValueError("into_weights without into: in place the weights move within themselves")
        if into is not None and all(a.data_ptr() == b.data_ptr() for a, b in ((self.k, to.k), (self.v, to.v), (self.k_exp, to.k_exp), (self.v_exp, to.v_exp))):
            raise ValueError("into lies in this cache's place: leave it out, so that the weights move with their rows")
        if not (0 < keep <= to.ctx) or first < 0 or recent < 0 or first + recent > keep:
            raise ValueError(f"keep {keep}, first {first}, recent {recent}: wanted first + recent <= keep <= {to.ctx}")
        batch = kv_len.numel()
        self._batch(batch, slot)
        to._batch(batch, slot)
        w = self._weights(weights, "weights")
        kept = torch.empty(batch, self.kv_heads, keep, dtype=_I32, device=self.device)
        length = torch.empty(batch, dtype=_I32, device=self.device)
        a = _lib.MdKv8EvictArgs(w, w if into is None else to._weights(into_weights, "into_weights"), self._per_sequence(slot, "slot", batch),
                                self._per_sequence(kv_len, "kv_len", batch), length.data_ptr(), kept.data_ptr(), batch, keep, first, recent)
        _launch(self._index, "md_kv8_evict", self._lib.md_kv8_evict, self._ref, to._ref, C.byref(a))
        return kept, length
