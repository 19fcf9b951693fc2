"""Rows of many tensors at once: fork, free and close the gaps.

The model's tensors and both moments of its optimiser share their first dimension, one row of each per Gaussian.
Refinement (``scene/gaussian_model.py:258-403``) copies some rows, makes new ones and removes others; the reference does
that tensor by tensor with concatenations and boolean masks.  Here one HIP launch (``gsr_select_rows``) moves the rows of
all tensors, and another (``gsr_keep_rows``) finds the kept ones.  There is no CPU path here, and no gradient flows
through these copies: they change what an optimiser works on, between its steps.
"""
from __future__ import annotations

import ctypes as C
import itertools
import math
import struct
from typing import List, Optional, Sequence, Tuple

import torch

import diff_gaussian_rasterization as _dgr

_lib = _dgr._lib
_lib.gsr_keep_rows_bytes.restype = C.c_size_t
_lib.gsr_keep_rows_bytes.argtypes = []
_lib.gsr_keep_rows.argtypes = [C.c_uint64, C.c_void_p, C.c_void_p, C.c_void_p, C.c_uint32, C.c_void_p, C.c_size_t, C.c_void_p]
_lib.gsr_select_rows.argtypes = [C.c_int, C.c_void_p, C.c_uint64, C.c_uint64, C.c_uint64, C.c_void_p, C.c_int, C.c_void_p]
MAX_ROWS = 0x7FFF0000                  # row numbers are 32-bit


def _checked(tensors: Sequence[torch.Tensor]) -> Tuple[List[torch.Tensor], torch.device, int]:
    tensors = list(tensors)
    if not tensors:
        raise ValueError("no tensors given")
    if {t.layout for t in tensors} != {torch.strided} or not all(t.is_cuda for t in tensors):
        raise ValueError("rows are moved between dense tensors on the GPU, got "
                         f"{[(str(t.layout), str(t.device)) for t in tensors][:8]}")
    if len({t.get_device() for t in tensors}) > 1:
        raise ValueError(f"tensors are on {sorted({str(t.device) for t in tensors})}: one call works on one GPU")
    shapes = [t.shape for t in tensors]
    rows = {s[0] if s else -1 for s in shapes}
    if len(rows) > 1 or -1 in rows:
        raise ValueError(f"tensors must share their first dimension, got shapes {[tuple(s) for s in shapes]}")
    rows = rows.pop()
    if rows > MAX_ROWS:
        raise ValueError(f"{rows} rows: at most {MAX_ROWS}")
    return tensors, tensors[0].device, rows


def _contiguous(tensors: Sequence[Optional[torch.Tensor]]) -> List[Optional[torch.Tensor]]:
    """Rows whose bytes are the values: in order, without gaps, and no conjugation or sign left for later."""
    if any(t is not None and (t.is_conj() or t.is_neg()) for t in tensors):
        tensors = [None if t is None else t.detach().resolve_conj().resolve_neg() for t in tensors]
    return [t if t is None or t.is_contiguous() else t.detach().contiguous() for t in tensors]


class _Move:
    """A move of rows, as far as it can be prepared before the number of rows is known; ``to`` launches it.
    ``tensors`` and ``appended`` are ``_contiguous``."""

    def __init__(self, tensors: List[torch.Tensor], appended: List[Optional[torch.Tensor]], rows: int, extra: int):
        self.tensors, self.appended = tensors, appended                               # kept alive until the launch
        self.tails = [t.shape[1:] for t in self.tensors]
        self.fixed = [(t.data_ptr(), 0 if e is None else e.data_ptr(), math.prod(s) * t.element_size())
                      for t, e, s in zip(self.tensors, self.appended, self.tails)]
        self.rows, self.extra = rows, extra

    def to(self, index: torch.Tensor, count: int) -> List[torch.Tensor]:
        out = [t.new_empty((count, *s)) for t, s in zip(self.tensors, self.tails)]
        if count:
            words = [w for (t, e, row), o in zip(self.fixed, out) for w in (t, e, o.data_ptr(), row)]
            _dgr._run("select_rows", _lib.gsr_select_rows, len(out), struct.pack(f"{len(words)}Q", *words), self.rows,
                      self.extra, count, index.data_ptr(), index.element_size(), _dgr._raw_stream(index.get_device()))
        return out


def select_rows(tensors: Sequence[torch.Tensor], index: torch.Tensor) -> List[torch.Tensor]:
    """``[t[index] for t in tensors]`` in one launch: new tensors whose row j is row ``index[j]`` of the old ones.

    ``tensors``: any types and row shapes on one GPU, the same number of rows.  ``index``: int32 or int64, one
    dimension, in any order and with repeats (a fork).  An index outside the rows, -1 for one, gives a row of zeros."""
    tensors, dev, rows = _checked(tensors)
    if index.dtype not in (torch.int32, torch.int64) or index.dim() != 1:
        raise TypeError(f"index must be a one-dimensional int32 or int64 tensor, got {index.dtype} of shape {tuple(index.shape)}")
    if index.device != dev:
        raise ValueError(f"index is on {index.device}, the tensors are on {dev}")
    count = index.numel()
    if count > MAX_ROWS:
        raise ValueError(f"{count} rows: at most {MAX_ROWS}")
    with _dgr._on_device(dev.index):
        return _Move(_contiguous(tensors), [None] * len(tensors), rows, 0).to(index.contiguous(), count)


_tickets = itertools.count(1)


def _landing(dev: torch.device):
    """This thread's pinned word for ``dev`` that a count of kept rows lands in: (the tensor that owns it, the word)."""
    slots = _dgr._per_device(dev)
    if "kept_rows" not in slots:
        word = torch.zeros((1,), dtype=torch.int64, pin_memory=True)
        slots["kept_rows"] = word, C.c_uint64.from_address(word.data_ptr())
    return slots["kept_rows"]


def _await_count(word: C.c_uint64, ticket: int, dev: torch.device) -> int:
    """The count that lands in ``word`` with ``ticket``.  Looks for it for a millisecond or two, which saves the wait
    for a copy to the host (13 us); a stream with more work than that before it is waited for."""
    for _ in range(10_000):
        value = word.value
        if value >> 32 == ticket:
            return value & 0xFFFFFFFF
    torch.cuda.current_stream(dev).synchronize()
    value = word.value
    if value >> 32 != ticket:
        raise RuntimeError("libgsr_hip keep_rows failed: the number of kept rows never arrived")
    return value & 0xFFFFFFFF


def _checked_compaction(tensors: Sequence[torch.Tensor], keep: torch.Tensor, appended: Optional[Sequence[Optional[torch.Tensor]]]):
    tensors, dev, rows = _checked(tensors)
    if keep.dtype != torch.bool or keep.dim() != 1:
        raise TypeError(f"keep must be a one-dimensional bool tensor, got {keep.dtype} of shape {tuple(keep.shape)}")
    if keep.device != dev:
        raise ValueError(f"keep is on {keep.device}, the tensors are on {dev}")
    total = keep.numel()
    extra = total - rows
    if extra < 0 or (extra and appended is None) or total > MAX_ROWS:
        raise ValueError(f"keep has {total} entries for {rows} rows" + (" and nothing appended" if appended is None else ""))
    more = [None] * len(tensors) if appended is None else list(appended)
    if len(more) != len(tensors):
        raise ValueError(f"{len(more)} appended entries for {len(tensors)} tensors")
    for t, e in zip(tensors, more):
        if e is not None and (e.shape != (extra, *t.shape[1:]) or e.dtype != t.dtype or e.device != dev or e.layout != torch.strided):
            raise ValueError(f"appended rows of shape {tuple(e.shape)}, {e.dtype} on {e.device} do not fit {extra} rows of a "
                             f"tensor of shape {tuple(t.shape)}, {t.dtype} on {dev}")
    return tensors, more, dev, rows, extra


def _again(tensors: Sequence[torch.Tensor], index: torch.Tensor, appended: Sequence[Optional[torch.Tensor]], extra: int) -> List[torch.Tensor]:
    """The rows of more ``tensors`` that a ``compact_rows`` with the same numbers of rows kept; arguments have been checked."""
    with _dgr._on_device(index.get_device()):
        return _Move(_contiguous(tensors), _contiguous(appended), tensors[0].shape[0], extra).to(index, index.numel())


def compact_rows(tensors: Sequence[torch.Tensor], keep: torch.Tensor,
                 appended: Optional[Sequence[Optional[torch.Tensor]]] = None) -> Tuple[List[torch.Tensor], torch.Tensor]:
    """``([torch.cat((t, a))[keep] for t, a in zip(tensors, appended)], index)`` without the concatenations.

    ``keep``: one bool per row, first the tensors' rows, then the appended ones.  ``appended``: for each tensor the rows
    behind its own, or None for rows of zeros (the moments of new Gaussians); None altogether: nothing is appended.
    ``index`` (int32): the positions of the kept rows, so ``index[j]`` is where row j of the results came from.
    The order stays.  The number of kept rows sizes the results, so the host waits for it and the call cannot be
    captured into a graph."""
    tensors, more, dev, rows, extra = _checked_compaction(tensors, keep, appended)
    total = rows + extra
    with _dgr._on_device(dev.index):
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("compact_rows reads the number of kept rows and cannot be captured into a graph; select_rows can")
        keep, tensors, more = keep.contiguous(), _contiguous(tensors), _contiguous(more)
        nb = _lib.gsr_keep_rows_bytes()
        scratch = torch.empty((nb,), dtype=torch.uint8, device=dev)
        index = torch.empty((total,), dtype=torch.int32, device=dev)
        _, word = _landing(dev)
        ticket = next(_tickets) & 0xFFFFFFFF or next(_tickets) & 0xFFFFFFFF       # never 0
        try:
            _dgr._run("keep_rows", _lib.gsr_keep_rows, total, keep.data_ptr(), index.data_ptr(), C.addressof(word), ticket,
                      scratch.data_ptr(), nb, _dgr._raw_stream(dev.index))
            move = _Move(tensors, more, rows, extra)                              # while the GPU counts
            count = _await_count(word, ticket, dev)
        except BaseException:
            # the count may still be under way: it must not land in a later call's word, nor in one that is gone
            torch.cuda.current_stream(dev).synchronize()
            raise
        index = index[:count]
        return move.to(index, count), index
