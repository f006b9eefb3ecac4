"""Bindings of the "kv8" kernel library (csrc/kv8_store.cu, kv8_attention.cu): a paged cache in 8 bits and the attention
over it.

``Pages`` holds e4m3 numbers and one scale, a power of two, per (page, kv head): an entry stands for number * |scale|.  A
page's scale is the smallest 2^e, -64 <= e <= 50, that holds its rows' largest magnitude within 448.  It begins anew when a
page gets its first row and only grows from there; when it grows, the rows that the page holds are rounded again.  A
magnitude is off by at most half a step of e4m3, 2^-4 of it, and by 2^-10 of the scale below 2^-6 scales (a growing scale may
add as much again there).  What is not finite, or above 448 * 2^50, is stored as NaN and makes the scale negative; it stays
with the rows that see it.  Scales are the store's to write: the attention takes them to be such powers of two.

Both operations take the engine's ``StepState``: which requests a step has, where each begins, how much it brings and how
much it holds already.  As everywhere in this package a step's metadata (its int32 tensors and the block table) lies in place
before the kernel in front of the call begins: kernels read it ahead of what that kernel writes.
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

import torch

from . import BF16, F32, _STATUS, _f32vec, _launched, _need_cuda, _rotary_table, _rows, device_status, dtype_code, raw_stream
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
        self.device, self.index = k.device, k.get_device()
        self.addresses = (k.data_ptr(), v.data_ptr(), k_scales.data_ptr(), v_scales.data_ptr())

    def tensors(self) -> tuple:
        return self.k, self.v, self.k_scales, self.v_scales

    def dequantized(self) -> tuple:
        """(keys, values) in float32, for looking at (computed with tensor operations)."""
        return tuple(t.to(torch.float32) * s.abs()[:, :, None, None] for t, s in ((self.k, self.k_scales), (self.v, self.v_scales)))


def check_head_dim(head_dim: int) -> None:
    if head_dim % 8 or not 8 <= head_dim <= MAX_HEAD_DIM:
        raise KernelError(f"an 8-bit cache holds heads of a multiple of 8 entries up to {MAX_HEAD_DIM}, not {head_dim}")


def _run():
    run = _FN["run"] = library(LIBRARY).gb_kv8_run
    run.argtypes, run.restype = [ctypes.c_char_p], ctypes.c_int
    return run


def _call(operation: int, index: int, device: torch.device, a, f0: float, step, part=None) -> None:
    n, r, longest = step.n_tokens, step.n_requests, step.max_q_len
    ws, splits, bias = 0, 0, 0
    if part is not None:
        ws, splits, bias = part.ws.data_ptr(), part.ws.shape[0], 0 if part.bias is None else part.bias.data_ptr()
    status = _STATUS.get(index)
    rc = (_FN.get("run") or _run())(
        _WORDS.pack(operation, raw_stream(device), (device_status(device) if status is None else status).data_ptr(), n, r, 0, longest,
                    step.max_ctx_len, 1 if longest == 1 and n == r else 0, 0, 0, 0, step.q_start.data_ptr(), step.q_len.data_ptr(),
                    step.start_pos.data_ptr(), ws, splits, bias, f0, *a))
    if rc < 0:
        check(library(LIBRARY), rc)
    _launched(rc)


_I32, _F32, _BF16 = torch.int32, torch.float32, torch.bfloat16


def _is(ok: bool, message: str) -> None:
    if not ok:
        raise KernelError(message)


# The checks of a call are made twice over: as one expression, which is what a good call costs (a decode step makes a dozen of
# them), and one by one with their messages where that expression is false.

def _step_ok(step, block_table, table, page_size: int, rows: int, index: int) -> bool:
    n, a, b, c = step.n_requests, step.q_start, step.q_len, step.start_pos
    return (a.dtype is _I32 and b.dtype is _I32 and c.dtype is _I32 and a.get_device() == index and b.get_device() == index
            and c.get_device() == index and a.is_contiguous() and b.is_contiguous() and c.is_contiguous() and a.numel() >= n
            and b.numel() >= n and c.numel() >= n and block_table.dtype is _I32 and block_table.get_device() == index
            and len(table) == 2 and block_table.is_contiguous() and table[0] >= n and rows >= step.n_tokens
            and table[1] * page_size >= step.max_ctx_len)


def _refuse_step(step, block_table, page_size: int, rows: int, index: int, what: str) -> None:
    n = step.n_requests
    for t in (step.q_start, step.q_len, step.start_pos):
        _is(t.dtype is _I32 and t.get_device() == index and t.is_contiguous() and t.numel() >= n,
            f"{what}: q_start, q_len and start_pos are {n} contiguous int32 values on cuda:{index}")
    _is(block_table.dtype is _I32 and block_table.get_device() == index and block_table.dim() == 2 and block_table.is_contiguous()
        and block_table.shape[0] >= n, f"{what}: the block table is contiguous int32 [{n} requests, entries] on cuda:{index}")
    _is(rows >= step.n_tokens, f"{what}: {rows} rows, the step has {step.n_tokens} tokens")
    _is(block_table.shape[1] * page_size >= step.max_ctx_len,
        f"{what}: block tables of {block_table.shape[1]} pages of {page_size} do not hold contexts of {step.max_ctx_len}")


def _vector_ok(t, n: int, index: int) -> bool:
    return t is None or (t.dtype is _F32 and t.is_contiguous() and t.numel() == n and t.get_device() == index)


def qk_norm_rope_store(qkv, q_out: torch.Tensor, heads: int, kv_heads: int, head_dim: int, q_gain: Optional[torch.Tensor],
                       k_gain: Optional[torch.Tensor], eps: float, inv_freq: Optional[torch.Tensor], rotary_dim: int,
                       adjacent_pairs: bool, step, block_table: torch.Tensor, pages: Optional[Pages]) -> torch.Tensor:
    """As ``ops.qk_norm_rope_store`` over an 8-bit cache: per-head RMSNorm (with gains) and rotation of q and k; q goes to
    ``q_out`` [tokens, heads * head_dim], k and v into their pages.  ``qkv``: rows [q heads | k heads | v heads], or the
    ``ops.Partials`` of their product.  ``inv_freq``: rotary_dim / 2 frequencies, or those and the factor on cosines and sines
    behind them.  ``pages`` None: rows of q alone (a layer that reads another layer's cache).  Only rows of the step's tokens
    are read or written.  A step writes to pages that no other request of it holds."""
    part = None if isinstance(qkv, torch.Tensor) else qkv
    x = qkv if part is None else part.ws
    index, cols = x.get_device(), (heads + (2 * kv_heads if pages is not None else 0)) * head_dim
    if inv_freq is not None and inv_freq.numel() != rotary_dim // 2 + 1 and not rotary_dim % 2:
        inv_freq = _rotary_table(inv_freq, rotary_dim)
    table, outs = block_table.shape, q_out.shape
    if part is None:
        shape, stride = x.shape, x.stride()
        good = len(shape) == 2 and (stride[1] == 1 or shape[1] == 1) and shape[1] >= cols and (x.dtype is _BF16 or x.dtype is _F32)
        rows, ld, dtype = shape[0], stride[0], x.dtype
    else:
        rows, ld, dtype = step.n_tokens, cols, _BF16
        good = (x.dtype is _F32 and x.is_contiguous() and x.dim() == 3 and tuple(x.shape[1:]) == (rows, cols)
                and part.dtype is _BF16 and _vector_ok(part.bias, cols, index))
    if not (good and index >= 0 and heads > 0 and kv_heads > 0 and not head_dim % 8 and 8 <= head_dim <= MAX_HEAD_DIM
            and q_out.dtype is dtype and q_out.get_device() == index and len(outs) == 2 and outs[1] == heads * head_dim
            and outs[0] >= step.n_tokens and q_out.is_contiguous() and _vector_ok(q_gain, head_dim, index)
            and _vector_ok(k_gain, head_dim, index) and (inv_freq is None or (
                not rotary_dim % 2 and 0 <= rotary_dim <= head_dim and _vector_ok(inv_freq, rotary_dim // 2 + 1, index)))
            and (pages is None or (pages.kv_heads == kv_heads and pages.head_dim == head_dim and pages.index == index))
            and _step_ok(step, block_table, table, 1 << 40 if pages is None else pages.page_size, rows, index)):
        _refuse_store(x, part, good, rows, cols, q_out, heads, kv_heads, head_dim, q_gain, k_gain, inv_freq, rotary_dim, step,
                      block_table, pages, index, dtype)
    if pages is not None:
        k, v, ks, vs = pages.addresses
        n_pages, page_size = pages.n_pages, pages.page_size
    else:
        k = v = ks = vs = n_pages = 0
        page_size = 16
    _call(0, index, x.device, (
        x.data_ptr() if part is None else 0, ld, BF16 if dtype is _BF16 else F32, q_out.data_ptr(),
        0 if q_gain is None else q_gain.data_ptr(), 0 if k_gain is None else k_gain.data_ptr(),
        0 if inv_freq is None else inv_freq.data_ptr(), 0 if inv_freq is None else rotary_dim, 1 if adjacent_pairs else 0, k, v, ks,
        vs, n_pages, page_size, heads, kv_heads, head_dim, block_table.data_ptr(), table[1]), eps, step, part)
    return q_out


def _refuse_store(x, part, good, rows, cols, q_out, heads, kv_heads, head_dim, q_gain, k_gain, inv_freq, rotary_dim, step, block_table,
                  pages, index, dtype) -> None:
    _need_cuda(x, q_out, q_gain, k_gain, inv_freq, block_table)
    _is(heads > 0 and kv_heads > 0, f"kv8 store: {heads} heads, {kv_heads} kv heads")
    check_head_dim(head_dim)
    if part is None:
        dtype_code(x.dtype)
        _is(good, f"kv8 store: rows of {cols} contiguous columns expected, got {tuple(x.shape)} strides {x.stride()}")
    _is(good, f"kv8 store: partial tiles [splits, {rows}, {cols}] float32 of a bfloat16 product expected")
    _is(q_out.dtype is dtype and q_out.dim() == 2 and q_out.shape[1] == heads * head_dim and q_out.shape[0] >= step.n_tokens
        and q_out.is_contiguous(), f"kv8 store: q_out is contiguous {dtype} [tokens, {heads * head_dim}]")
    _f32vec(q_gain, head_dim, "q gain"), _f32vec(k_gain, head_dim, "k gain")
    _is(inv_freq is None or (not rotary_dim % 2 and 0 <= rotary_dim <= head_dim), f"kv8 store: a rotation over {rotary_dim} of {head_dim} entries")
    _f32vec(inv_freq, rotary_dim // 2 + 1, "rotary table")
    _is(pages is None or (pages.kv_heads, pages.head_dim, pages.index) == (kv_heads, head_dim, index),
        "kv8 store: the pages hold another number of kv heads, other heads, or lie on another device")
    _refuse_step(step, block_table, 1 << 40 if pages is None else pages.page_size, rows, index, "kv8 store")
    raise KernelError(f"kv8 store: all tensors lie on cuda:{index}")


def paged_attention(q: torch.Tensor, heads: int, kv_heads: int, head_dim: int, pages: Pages, block_table: torch.Tensor,
                    scale: float, window: int, out: torch.Tensor, step) -> torch.Tensor:
    """out[t, h, :] = softmax over visible keys of (q.K)*scale, times V, over an 8-bit cache; q may be a column slice of a
    wider row.  ``scale``: finite, of any sign.  ``window`` 0: none; block tables hold the step's longest context.  Rows of
    ``out`` behind the step's tokens are left as they are."""
    index, cols, qs, os_, dtype = q.get_device(), heads * head_dim, q.stride(), out.stride(), q.dtype
    table, rows, outs = block_table.shape, q.shape, out.shape
    if not (index >= 0 and heads > 0 and kv_heads > 0 and not heads % kv_heads and len(qs) == 2 and len(os_) == 2
            and rows[1] == cols and outs[1] == cols and (qs[1] == 1 or cols == 1) and (os_[1] == 1 or cols == 1)
            and out.dtype is dtype and (dtype is _BF16 or dtype is _F32) and outs[0] >= step.n_tokens and out.get_device() == index
            and pages.kv_heads == kv_heads and pages.head_dim == head_dim and pages.index == index and window is not None and window >= 0
            and (os_[0] >= cols or outs[0] == 1) and _step_ok(step, block_table, table, pages.page_size, rows[0], index)):
        _refuse_attention(q, heads, kv_heads, head_dim, pages, block_table, window, out, step, index)
    k, v, ks, vs = pages.addresses
    _call(1, index, q.device, (q.data_ptr(), qs[0], BF16 if dtype is _BF16 else F32, out.data_ptr(), os_[0], k, v, ks, vs, pages.n_pages,
                               pages.page_size, heads, kv_heads, head_dim, block_table.data_ptr(), table[1], window, 0, 0, 0),
          scale, step)
    return out


def _refuse_attention(q, heads, kv_heads, head_dim, pages, block_table, window, out, step, index) -> None:
    _need_cuda(q, out, block_table)
    _is(heads > 0 and kv_heads > 0 and not heads % kv_heads, f"kv8 attention: {heads} heads are not a multiple of {kv_heads} kv heads")
    dtype_code(q.dtype)
    _is(q.dim() == 2 and out.dim() == 2 and q.shape[1] == out.shape[1] == heads * head_dim and q.dtype is out.dtype
        and out.shape[0] >= step.n_tokens, f"kv8 attention: q and out are [tokens, {heads * head_dim}] of one dtype")
    _rows(q, "kv8 attention q"), _rows(out, "kv8 attention out")
    _is((pages.kv_heads, pages.head_dim, pages.index) == (kv_heads, head_dim, index) and out.get_device() == index,
        f"kv8 attention: the pages hold {pages.kv_heads} kv heads of {pages.head_dim} on {pages.device}")
    _is(window is not None and window >= 0, f"kv8 attention: a window of {window} keys (0: none)")
    _is(out.stride(0) >= out.shape[1] or out.shape[0] == 1, "kv8 attention: rows of out lie over one another")
    _refuse_step(step, block_table, pages.page_size, q.shape[0], index, "kv8 attention")
    raise KernelError("kv8 attention: a call of these tensors is not taken")
