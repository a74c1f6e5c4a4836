"""Beam search on the device: the choice among all beams' continuations, and the beams' states moved behind their parents.

    choice = select_beams(logits, scores, ended=ended, end_id=eos)     # [batch * beams, vocab] -> tokens, parents, scores, ended
    reorder_states([k_slab, v_slab], choice.parents, slot_dim=1)       # the caches of all layers, in place

A search starts with all scores but the first of every input -inf: the first step then takes the best tokens of one beam.  Both run on the
current stream of their tensors' device, allocate through torch only, never synchronise and can be captured into a graph.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple, Optional, Sequence

import torch

from . import _lib
from .block_cache import _launch, _need

MAX_BEAMS = _lib.MD_MAX_BEAMS
_DTYPES = {torch.bfloat16: _lib.MD_DTYPE_BF16, torch.float32: _lib.MD_DTYPE_F32}


class BeamChoice(NamedTuple):
    tokens: torch.Tensor   # int32 [batch, beams]
    parents: torch.Tensor  # int32 [batch, beams]: the beam, of the same input, that the token goes on from
    scores: torch.Tensor   # fp32 [batch, beams], falling (by rank)
    ended: torch.Tensor    # int32 [batch, beams]


def _gpu(t: torch.Tensor, what: str) -> torch.device:
    if t.device.type != "cuda":
        raise _lib.MoondreamHipError(f"{what} needs a GPU device; there is no CPU path")
    return t.device


def select_beams(logits: torch.Tensor, scores: torch.Tensor, ended: Optional[torch.Tensor] = None, end_id: int = -1, suppress_id: int = -1,
                 rank_weight: Optional[torch.Tensor] = None) -> BeamChoice:
    """The ``beams`` best continuations of every input's beams.  ``logits`` [batch * beams, vocab] (bf16 or fp32, rows may lie apart), ``scores`` fp32
    [batch, beams]: a beam's sum of log probabilities so far, -inf for one that does not exist.  ``ended`` (int32 [batch, beams]): beams that have ended
    stay in the running with their score, as one continuation ``end_id``.  ``rank_weight`` (fp32 [batch, beams], > 0) multiplies the totals of a beam's
    continuations for the choice alone (a length penalty: 1 / length ** alpha).  Ties: the lower beam, the larger logit, the lower token.
    Where fewer than ``beams`` continuations are left: token ``end_id``, score -inf, ended, its own parent."""
    if scores.dim() != 2 or logits.dim() != 2 or logits.shape[0] != scores.shape[0] * scores.shape[1] or logits.dtype not in _DTYPES or logits.shape[1] == 0:
        raise ValueError(f"logits {tuple(logits.shape)} {logits.dtype} for scores {tuple(scores.shape)}: wanted [batch * beams, vocab] bfloat16 or float32")
    batch, beams = scores.shape
    vocab = logits.shape[1]
    if not 2 <= beams <= MAX_BEAMS or batch == 0:
        raise ValueError(f"{batch} inputs of {beams} beams: wanted 2 to {MAX_BEAMS} beams")
    if end_id >= vocab or (end_id < 0 and ended is not None):
        raise ValueError(f"end_id {end_id} of {vocab} tokens" + (" with ended beams" if ended is not None else ""))
    if logits.stride(1) != 1 or logits.stride(0) < vocab:
        raise ValueError(f"logits of strides {logits.stride()}: rows have to be contiguous and apart")
    dev, shape = _gpu(logits, "select_beams"), (batch, beams)
    tokens, parents, stop = torch.empty((3, batch, beams), dtype=torch.int32, device=dev).unbind(0)
    new = torch.empty(shape, dtype=torch.float32, device=dev)
    lib = _lib.load()
    need = lib.md_beam_workspace_bytes(batch, beams, vocab)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    at = tokens.data_ptr()
    a = _lib.MdBeamArgs(logits.data_ptr(), logits.stride(0), _DTYPES[logits.dtype], batch, beams, vocab, suppress_id, max(end_id, -1),
                        _need(scores, "scores", torch.float32, dev.index, shape), None if ended is None else _need(ended, "ended", torch.int32, dev.index, shape),
                        None if rank_weight is None else _need(rank_weight, "rank_weight", torch.float32, dev.index, shape),
                        at, at + 4 * batch * beams, new.data_ptr(), at + 8 * batch * beams, ws.data_ptr(), need)
    _launch(dev.index, "md_beam_select", lib.md_beam_select, C.byref(a))
    return BeamChoice(tokens, parents, new, stop)


@functools.lru_cache(maxsize=256)
def _runs(shape: tuple, stride: tuple, size: int, slot_dim: int, name: str):
    """(slot stride, outer count and stride, run count and stride, run length), in bytes, of the slots of a tensor of that layout."""
    dims = [(n, s * size) for d, (n, s) in enumerate(zip(shape, stride)) if d != slot_dim and n > 1]
    length = size
    while dims and dims[-1][1] == length:
        length *= dims.pop()[0]
    joined = []
    for n, s in dims:  # neighbours that are one dimension in memory
        if joined and joined[-1][1] == n * s:
            joined[-1] = (joined[-1][0] * n, s)
        else:
            joined.append((n, s))
    if len(joined) > 2:
        raise ValueError(f"{name}: strides {stride} leave more than two dimensions that lie apart")
    outer, segs = ([(1, 0)] * 2 + joined)[-2:]
    return stride[slot_dim] * size, outer, segs, length


def reorder_states(states: Sequence[torch.Tensor], parents: torch.Tensor, into: Optional[Sequence[torch.Tensor]] = None, slot_dim: int = 0) -> None:
    """Slot b * beams + k of every state <- its slot b * beams + parents[b, k] (``parents``: int32 [batch, beams]), in place, or from ``states`` to ``into``
    (tensors of the same shapes and types that share no memory with them).  ``slot_dim``: the states' dimension of slots; the first batch * beams
    slots take part.  States may be views -- the rows of an answer in all layers' slabs, ``slab[:, :, :, first:last]`` -- whose dimensions
    besides the slots' make at most two strides apart; no two of them share memory, nor does one that is written with another that is read.  What lies in front of the answers is the same for all beams of an input and need not be moved."""
    if parents.dim() != 2 or not 1 <= parents.shape[1] <= MAX_BEAMS or parents.shape[0] == 0:
        raise ValueError(f"parents {tuple(parents.shape)}: wanted [batch, 1 to {MAX_BEAMS} beams]")
    batch, beams = parents.shape
    into = states if into is None else into
    if len(into) != len(states):
        raise ValueError(f"{len(states)} states into {len(into)}")
    parts = []
    for i, (src, dst) in enumerate(zip(states, into)):
        name, shape, stride, size = f"state {i}", src.shape, src.stride(), src.element_size()
        if shape != dst.shape or src.dtype is not dst.dtype or src.device != parents.device or dst.device != parents.device:
            raise ValueError(f"{name}: {tuple(shape)} {src.dtype} on {src.device} into {tuple(dst.shape)} {dst.dtype} on {dst.device}")
        n = len(shape)
        if not -n <= slot_dim < n or shape[slot_dim] < batch * beams:
            raise ValueError(f"{name}: {tuple(shape)} has fewer than {batch * beams} slots in dimension {slot_dim}")
        if src.numel() == 0:
            continue
        a = _runs(tuple(shape), stride, size, slot_dim % n, name)
        b = a if dst is src else _runs(tuple(shape), dst.stride(), size, slot_dim % n, name)
        if (a[1][0], a[2][0], a[3]) != (b[1][0], b[2][0], b[3]):
            raise ValueError(f"{name}: strides {stride} into {dst.stride()}")
        parts.append((src.data_ptr(), dst.data_ptr(), a[0], b[0], a[1][1], b[1][1], a[2][1], b[2][1], a[3], a[1][0], a[2][0]))
    if not parts:
        return
    dev = _gpu(parents, "reorder_states")
    _launch(dev.index, "md_state_reorder", _lib.load().md_state_reorder, (_lib.MdStatePart * len(parts))(*parts), len(parts),
            _need(parents, "parents", torch.int32, dev.index, (batch, beams)), batch, beams)
