"""Rows of many tensors at once: fork, free and close the gaps.

The model's tensors and both moments of its optimiser share their first dimension, one row of each per Gaussian.
Refinement (``scene/gaussian_model.py:258-403``) copies some rows, makes new ones and removes others; the reference does
that tensor by tensor with concatenations and boolean masks.  Here one HIP launch (``gsr_select_rows``) moves the rows of
all tensors, and another (``gsr_keep_rows``) finds the kept ones.  There is no CPU path here, and no gradient flows
through these copies: they change what an optimiser works on, between its steps.
"""
from __future__ import annotations

import ctypes as C
from typing import List, Optional, Sequence, Tuple

import torch

import diff_gaussian_rasterization as _dgr

_lib = _dgr._lib
_lib.gsr_keep_rows_bytes.restype = C.c_size_t
_lib.gsr_keep_rows_bytes.argtypes = []
_lib.gsr_keep_rows.argtypes = [C.c_uint64, C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t, C.c_void_p]
_lib.gsr_select_rows.argtypes = [C.c_int, C.c_void_p, C.c_uint64, C.c_uint64, C.c_uint64, C.c_void_p, C.c_int, C.c_void_p]
MAX_ROWS = 0x7FFF0000                  # row numbers are 32-bit


def _checked(tensors: Sequence[torch.Tensor]) -> Tuple[List[torch.Tensor], torch.device, int]:
    tensors = list(tensors)
    if not tensors:
        raise ValueError("no tensors given")
    dev, rows = tensors[0].device, tensors[0].shape[0] if tensors[0].dim() else -1
    for t in tensors:
        if not t.is_cuda or t.layout != torch.strided:
            raise ValueError(f"rows are moved between dense tensors on the GPU, got {t.layout} on {t.device}")
        if t.device != dev:
            raise ValueError(f"tensors are on {dev} and {t.device}: one call works on one GPU")
        if t.dim() == 0 or t.shape[0] != rows:
            raise ValueError(f"tensors must share their first dimension, got shapes {[tuple(x.shape) for x in tensors]}")
    if rows > MAX_ROWS:
        raise ValueError(f"{rows} rows: at most {MAX_ROWS}")
    return tensors, dev, rows


def _move(tensors: List[torch.Tensor], appended: List[Optional[torch.Tensor]], rows: int, extra: int, index: torch.Tensor,
          count: int) -> List[torch.Tensor]:
    out, words, hold = [], [], []
    for t, e in zip(tensors, appended):
        o = torch.empty((count,) + t.shape[1:], dtype=t.dtype, device=t.device)
        t = t.contiguous()
        e = None if e is None else e.contiguous()
        hold.append((t, e))
        out.append(o)
        row = t.element_size()
        for s in t.shape[1:]:
            row *= s
        words += (t.data_ptr(), 0 if e is None else e.data_ptr(), o.data_ptr(), row)
    _dgr._run("select_rows", _lib.gsr_select_rows, len(out), (C.c_uint64 * len(words))(*words), rows, extra, count,
              _dgr._ptr(index), index.element_size(), _dgr._stream())
    return out


@torch.no_grad()
def select_rows(tensors: Sequence[torch.Tensor], index: torch.Tensor) -> List[torch.Tensor]:
    """``[t[index] for t in tensors]`` in one launch: new tensors whose row j is row ``index[j]`` of the old ones.

    ``tensors``: any types and row shapes on one GPU, the same number of rows.  ``index``: int32 or int64, one
    dimension, in any order and with repeats (a fork).  An index outside the rows, -1 for one, gives a row of zeros."""
    tensors, dev, rows = _checked(tensors)
    if index.dtype not in (torch.int32, torch.int64) or index.dim() != 1:
        raise TypeError(f"index must be a one-dimensional int32 or int64 tensor, got {index.dtype} of shape {tuple(index.shape)}")
    if index.device != dev:
        raise ValueError(f"index is on {index.device}, the tensors are on {dev}")
    if index.numel() > MAX_ROWS:
        raise ValueError(f"{index.numel()} rows: at most {MAX_ROWS}")
    with torch.cuda.device(dev):
        return _move(tensors, [None] * len(tensors), rows, 0, index.contiguous(), index.numel())


@torch.no_grad()
def compact_rows(tensors: Sequence[torch.Tensor], keep: torch.Tensor,
                 appended: Optional[Sequence[Optional[torch.Tensor]]] = None) -> Tuple[List[torch.Tensor], torch.Tensor]:
    """``([torch.cat((t, a))[keep] for t, a in zip(tensors, appended)], index)`` without the concatenations.

    ``keep``: one bool per row, first the tensors' rows, then the appended ones.  ``appended``: for each tensor the rows
    behind its own, or None for rows of zeros (the moments of new Gaussians); None altogether: nothing is appended.
    ``index`` (int32): the positions of the kept rows, so ``index[j]`` is where row j of the results came from.
    The order stays.  The number of kept rows sizes the results, so the call waits for the GPU once."""
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
        if e is not None and (e.shape != (extra,) + t.shape[1:] or e.dtype != t.dtype or e.device != dev or e.layout != torch.strided):
            raise ValueError(f"appended rows of shape {tuple(e.shape)}, {e.dtype} on {e.device} do not fit {extra} rows of a "
                             f"tensor of shape {tuple(t.shape)}, {t.dtype} on {dev}")
    with torch.cuda.device(dev):
        keep = keep.contiguous()
        nb = _lib.gsr_keep_rows_bytes()
        scratch = torch.empty((nb,), dtype=torch.uint8, device=dev)
        index = torch.empty((total + 1,), dtype=torch.int32, device=dev)          # and the count behind them
        _dgr._run("keep_rows", _lib.gsr_keep_rows, total, _dgr._ptr(keep), _dgr._ptr(index),
                  C.c_void_p(index.data_ptr() + 4 * total), _dgr._ptr(scratch), nb, _dgr._stream())
        count = int(index[total])
        index = index[:count]
        return _move(tensors, more, rows, extra, index, count), index
