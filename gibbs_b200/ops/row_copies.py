"""Copies of rows within a cache's tensors (csrc/row_copies.cu): pages from one id to another, state slots likewise."""
from __future__ import annotations

import ctypes
import struct
from typing import Sequence

import torch

from . import _launched, raw_stream
from .library import KernelError, check, library

LIBRARY = "core"                 # (an engine forks whatever its cache is held in)
MAX_GROUPS = 16


class RowCopies:
    """Row copies within ``groups`` of tensors: the tensors of a group (K and V pages of every layer and their scales, say)
    have one number of rows, and what is copied in one is copied in all.  A tensor's rows are contiguous; the rows may be
    strided; groups share no memory.  Made once for a cache; holds the tensors."""

    def __init__(self, groups: Sequence[Sequence[torch.Tensor]]):
        self.groups = [list(g) for g in groups]
        if not 1 <= len(self.groups) <= MAX_GROUPS:
            raise KernelError(f"row copies: {len(self.groups)} groups of tensors, 1 to {MAX_GROUPS} expected")
        everything = [t for g in self.groups for t in g]
        if not everything or any(not t.is_cuda for t in everything) or len({t.device for t in everything}) != 1:
            raise KernelError("row copies: tensors on one CUDA device expected")
        self.device = everything[0].device
        lib = library(LIBRARY)
        most = lib.gb_row_copies_piece_bytes()
        records, n_pieces = [], []
        for i, g in enumerate(self.groups):
            if not g or any(t.dim() < 1 or t.shape[0] != g[0].shape[0] for t in g):
                raise KernelError(f"row copies: the tensors of group {i} have one number of rows")
            before = len(records)
            for t in g:
                if t.shape[0] == 0 or t[0].numel() == 0:
                    continue
                if not t[0].is_contiguous():
                    raise KernelError(f"row copies: rows of {tuple(t.shape[1:])} in group {i} are not contiguous")
                size, stride = t[0].numel() * t.element_size(), t.stride(0) * t.element_size()
                if t.shape[0] > 1 and stride < size:
                    raise KernelError(f"row copies: rows of group {i} overlap")
                records += [(t.data_ptr() + at, stride, min(most, size - at)) for at in range(0, size, most)]
            n_pieces.append(len(records) - before)
        self._pieces = torch.tensor(records or [(0, 0, 0)], dtype=torch.int64).to(self.device)
        n = len(self.groups)
        self._table, self._sizes = self._pieces.data_ptr(), [v for i, g in enumerate(self.groups) for v in (n_pieces[i], g[0].shape[0])]
        self._format = f"={3 + 4 * n}q"
        self._run = lib.gb_row_copies
        self._run.argtypes, self._run.restype = [ctypes.c_char_p], ctypes.c_int
        torch.cuda.current_stream(self.device).synchronize()       # the records lie in place whatever stream copies use

    def copy(self, pairs: Sequence) -> int:
        """``pairs``: for each group the (src, dst) rows, as a sequence of pairs or an int32 tensor [n, 2] on the host.  Every
        source is read as it was before the call; a row that is a destination twice, or a destination and a source, is
        refused, and then nothing is copied.  Launches on the current stream; returns the number of kernels."""
        if len(pairs) != len(self.groups):
            raise KernelError(f"row copies: pairs for {len(pairs)} groups, {len(self.groups)} expected")
        keep, words = [], []
        for i, p in enumerate(pairs):
            if isinstance(p, torch.Tensor):
                if p.is_cuda or p.dtype != torch.int32 or p.dim() != 2 or p.shape[1] != 2 or not p.is_contiguous():
                    raise KernelError(f"row copies: pairs of group {i} are contiguous int32 [n, 2] on the host")
                keep.append(p)
                words += (p.data_ptr(), len(p))
            else:
                try:
                    flat = [v for src, dst in p for v in (src, dst)]
                    a = (ctypes.c_int * len(flat)).from_buffer_copy(struct.pack(f"={len(flat)}i", *flat)) if flat else None
                except (struct.error, TypeError, ValueError) as e:
                    raise KernelError(f"row copies: pairs of group {i} are (src, dst), 32-bit integers ({e})") from None
                keep.append(a)
                words += (0 if a is None else ctypes.addressof(a), len(flat) // 2)
        rc = self._run(struct.pack(self._format, self._table, raw_stream(self.device), len(self.groups), *words, *self._sizes))
        if rc < 0:
            check(library(LIBRARY), rc)
        _launched(rc)
        return rc
