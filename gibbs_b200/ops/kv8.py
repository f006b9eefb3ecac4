"""Bindings of the "kv8" kernel library (csrc/kv8_store.cu, kv8_attention.cu): a paged cache in 8 bits and the attention
over it.

``Pages`` holds e4m3 numbers and one scale, a power of two, per (page, kv head): an entry stands for number * |scale|.  A
page's scale is the smallest 2^e, -64 <= e <= 50, that holds its rows' largest magnitude within 448.  It begins anew when a
page gets its first row and only grows from there; when it grows, the rows that the page holds are rounded again.  A
magnitude is off by at most half a step of e4m3, 2^-4 of it, and by 2^-10 of the scale below 2^-6 scales (a growing scale may
add as much again there).  What is not finite, or above 448 * 2^50, is stored as NaN and makes the scale negative; it stays
with the rows that see it.

Both operations take the engine's ``StepState``: which requests a step has, where each begins, how much it brings and how
much it holds already.  As everywhere in this package a step's metadata (its int32 tensors and the block table) lies in place
before the kernel in front of the call begins: kernels read it ahead of what that kernel writes.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

import torch

from . import _f32vec, _launched, _need_cuda, _rotary_table, _rows, device_status, dtype_code, raw_stream
from .library import KernelError, check, library

LIBRARY = "kv8"
OPERATIONS = ("kv8_store", "kv8_attention")
DTYPE = torch.float8_e4m3fn
TAKES_PARTIALS = 1 << 29         # a record's flag: the operation adds the partial tiles of the product in front
MAX_HEAD_DIM = 256

# what csrc/kv8_call.cu reads: operation, stream, status word, twelve symbols, partial tiles, their number and bias; the
# floating operand; twenty operands
_WORDS = struct.Struct("=18qd20q")

_FN: dict = {}
_IDS: dict = {}


def _function(name: str):
    fn = _FN.get(name)
    if fn is None:
        fn = _FN[name] = getattr(library(LIBRARY), "gb_op_" + name)
        fn.restype = ctypes.c_int
    return fn


def plan_id(name: str) -> int:
    """The operation's id with the step walker (registered at first use)."""
    i = _IDS.get(name)
    if i is None:
        from ..engine.plan import register_op
        i = _IDS[name] = register_op("kv8." + name, _function(name))
    return i


class Pages:
    """One entry's cache: ``k``, ``v`` e4m3 [n_pages, kv_heads, page_size, head_dim], ``k_scales``, ``v_scales`` float32
    [n_pages, kv_heads], all contiguous and on one device."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scales: torch.Tensor, v_scales: torch.Tensor):
        if k.dim() != 4 or k.dtype != DTYPE or not k.is_contiguous() or v.shape != k.shape or v.dtype != DTYPE \
                or not v.is_contiguous():
            raise KernelError("8-bit pages: keys and values are contiguous float8_e4m3fn [n_pages, kv_heads, page_size, head_dim] "
                              f"of one shape, got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
        for s in (k_scales, v_scales):
            if s.shape != k.shape[:2] or s.dtype != torch.float32 or not s.is_contiguous():
                raise KernelError(f"8-bit pages: scales are contiguous float32 {tuple(k.shape[:2])}, got {tuple(s.shape)} {s.dtype}")
        if len({t.device for t in (k, v, k_scales, v_scales)}) != 1:
            raise KernelError("8-bit pages: keys, values and scales lie on one device")
        self.n_pages, self.kv_heads, self.page_size, self.head_dim = k.shape
        check_head_dim(self.head_dim)
        if k.data_ptr() % 16 or v.data_ptr() % 16:
            raise KernelError("8-bit pages: keys and values begin at 16-byte boundaries")
        self.k, self.v, self.k_scales, self.v_scales = k, v, k_scales, v_scales
        self.device = k.device
        self.addresses = (k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr())

    def tensors(self) -> tuple:
        return self.k, self.v, self.k_scales, self.v_scales

    def dequantized(self) -> tuple:
        """(keys, values) in float32, for looking at (computed with tensor operations)."""
        return tuple(t.to(torch.float32) * s.abs()[:, :, None, None] for t, s in ((self.k, self.k_scales), (self.v, self.v_scales)))


def check_head_dim(head_dim: int) -> None:
    if head_dim % 8 or not 8 <= head_dim <= MAX_HEAD_DIM:
        raise KernelError(f"an 8-bit cache holds heads of a multiple of 8 entries up to {MAX_HEAD_DIM}, not {head_dim}")


def _call(operation: int, device: torch.device, a, f0: float, step, part=None) -> None:
    run = _FN.get("run")
    if run is None:
        run = _FN["run"] = library(LIBRARY).gb_kv8_run
        run.argtypes, run.restype = [ctypes.c_char_p], ctypes.c_int
    n, r, longest = step.n_tokens, step.n_requests, step.max_q_len
    ws, splits, bias = 0, 0, 0
    if part is not None:
        ws, splits, bias = part.ws.data_ptr(), part.ws.shape[0], 0 if part.bias is None else part.bias.data_ptr()
    rc = run(_WORDS.pack(operation, raw_stream(device), device_status(device).data_ptr(), n, r, 0, longest, step.max_ctx_len,
                         1 if longest == 1 and n == r else 0, 0, 0, 0, step.q_start.data_ptr(), step.q_len.data_ptr(),
                         step.start_pos.data_ptr(), ws, splits, bias, f0, *a))
    if rc < 0:
        check(library(LIBRARY), rc)
    _launched(rc)


_I32 = torch.int32


def _check_step(step, block_table: torch.Tensor, rows: int, device: torch.device, what: str) -> None:
    n = step.n_requests
    for t in (step.q_start, step.q_len, step.start_pos):
        if t.dtype is not _I32 or t.device != device or not t.is_contiguous() or t.numel() < n:
            raise KernelError(f"{what}: q_start, q_len and start_pos are {n} contiguous int32 values on {device}")
    if block_table.dtype is not _I32 or block_table.device != device or block_table.dim() != 2 \
            or not block_table.is_contiguous() or block_table.shape[0] < n:
        raise KernelError(f"{what}: the block table is contiguous int32 [{n} requests, entries] on {device}")
    if rows < step.n_tokens:
        raise KernelError(f"{what}: {rows} rows, the step has {step.n_tokens} tokens")


def qk_norm_rope_store(qkv, q_out: torch.Tensor, heads: int, kv_heads: int, head_dim: int, q_gain: Optional[torch.Tensor],
                       k_gain: Optional[torch.Tensor], eps: float, inv_freq: Optional[torch.Tensor], rotary_dim: int,
                       adjacent_pairs: bool, step, block_table: torch.Tensor, pages: Optional[Pages]) -> torch.Tensor:
    """As ``ops.qk_norm_rope_store`` over an 8-bit cache: per-head RMSNorm (with gains) and rotation of q and k; q goes to
    ``q_out`` [tokens, heads * head_dim], k and v into their pages.  ``qkv``: rows [q heads | k heads | v heads], or the
    ``ops.Partials`` of their product.  ``pages`` None: rows of q alone (a layer that reads another layer's cache).  Only
    rows of the step's tokens are read or written."""
    part = qkv if not isinstance(qkv, torch.Tensor) else None
    x = qkv if part is None else part.ws
    _need_cuda(x, q_out, q_gain, k_gain, inv_freq)
    if heads <= 0 or kv_heads <= 0:
        raise KernelError(f"kv8 store: {heads} heads, {kv_heads} kv heads")
    check_head_dim(head_dim)
    cols = (heads + (2 * kv_heads if pages is not None else 0)) * head_dim
    if part is not None:
        if x.dtype != torch.float32 or not x.is_contiguous() or x.dim() != 3 or x.shape[1:] != (step.n_tokens, cols) \
                or part.dtype != torch.bfloat16:
            raise KernelError(f"kv8 store: partial tiles [splits, {step.n_tokens}, {cols}] float32 of a bfloat16 product expected")
        _f32vec(part.bias, cols, "qkv bias")
        rows, ld, dtype = x.shape[1], cols, torch.bfloat16
    else:
        rows, ld, dtype = x.shape[0], _rows(x, "qkv"), x.dtype
        if x.shape[1] < cols:
            raise KernelError(f"kv8 store: rows of {x.shape[1]} columns, {cols} needed")
    code = dtype_code(dtype)
    if q_out.dtype != dtype or q_out.dim() != 2 or q_out.shape[1] != heads * head_dim or q_out.shape[0] < step.n_tokens \
            or not q_out.is_contiguous():
        raise KernelError(f"kv8 store: q_out is contiguous {dtype} [tokens, {heads * head_dim}]")
    _f32vec(q_gain, head_dim, "q gain"), _f32vec(k_gain, head_dim, "k gain")
    if inv_freq is not None and (rotary_dim % 2 or not 0 <= rotary_dim <= head_dim):
        raise KernelError(f"kv8 store: a rotation over {rotary_dim} of {head_dim} entries")
    table = _rotary_table(inv_freq, rotary_dim)
    _check_step(step, block_table, rows, x.device, "kv8 store")
    if pages is not None:
        if (pages.kv_heads, pages.head_dim) != (kv_heads, head_dim) or pages.device != x.device:
            raise KernelError(f"kv8 store: the pages hold {pages.kv_heads} kv heads of {pages.head_dim} on {pages.device}")
        k, v, ks, vs = pages.addresses
        n_pages, page_size = pages.n_pages, pages.page_size
    else:
        k = v = ks = vs = n_pages = 0
        page_size = 16
    a = (x.data_ptr() if part is None else 0, ld, code, q_out.data_ptr(), 0 if q_gain is None else q_gain.data_ptr(),
         0 if k_gain is None else k_gain.data_ptr(), 0 if table is None else table.data_ptr(), rotary_dim if table is not None else 0,
         1 if adjacent_pairs else 0, k, v, ks, vs, n_pages, page_size, heads, kv_heads, head_dim, block_table.data_ptr(),
         block_table.shape[1])
    _call(0, x.device, a, eps, step, part)
    return q_out


def paged_attention(q: torch.Tensor, heads: int, kv_heads: int, head_dim: int, pages: Pages, block_table: torch.Tensor,
                    scale: float, window: int, out: torch.Tensor, step) -> torch.Tensor:
    """out[t, h, :] = softmax over visible keys of (q.K)*scale, times V, over an 8-bit cache; q may be a column slice of a
    wider row.  Rows of ``out`` behind the step's tokens are left as they are."""
    _need_cuda(q, out)
    if heads <= 0 or kv_heads <= 0 or heads % kv_heads:
        raise KernelError(f"kv8 attention: {heads} heads are not a multiple of {kv_heads} kv heads")
    cols, device = heads * head_dim, q.device
    if q.dim() != 2 or out.dim() != 2 or q.shape[1] != cols or out.shape[1] != cols or q.dtype != out.dtype \
            or out.shape[0] < step.n_tokens:
        raise KernelError(f"kv8 attention: q and out are [tokens, {cols}] of one dtype")
    if pages.kv_heads != kv_heads or pages.head_dim != head_dim or pages.device != device or out.device != device:
        raise KernelError(f"kv8 attention: the pages hold {pages.kv_heads} kv heads of {pages.head_dim} on {pages.device}")
    if window is None or window < 0:
        raise KernelError(f"kv8 attention: a window of {window} keys (0: none)")
    _check_step(step, block_table, q.shape[0], device, "kv8 attention")
    k, v, ks, vs = pages.addresses
    _call(1, device, (q.data_ptr(), _rows(q, "q"), dtype_code(q.dtype), out.data_ptr(), _rows(out, "out"), k, v, ks, vs,
                      pages.n_pages, pages.page_size, heads, kv_heads, head_dim, block_table.data_ptr(), block_table.shape[1],
                      window, 0, 0, 0), scale, step)
    return out
