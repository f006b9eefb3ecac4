"""Sizes of an 8-bit cache that the host works out or refuses."""
import ctypes
import math
import struct
from types import SimpleNamespace

import pytest
import torch

from gibbs_b200.parts.base import PagedKV


@pytest.mark.parametrize("page,kv_heads,hd", [(16, 8, 64), (1, 4, 8), (5, 1, 16), (128, 2, 128)])
def test_pages_by_memory_count_the_scales(monkeypatch, page, kv_heads, hd):
    """What `pages_for` hands out fits the memory that it may take, with the scales of 8-bit pages, and one page more does not."""
    from gibbs_b200.cache import CacheManager
    from gibbs_b200.engine.api import pages_for
    needs = [([PagedKV(kv_heads, hd, in_8_bits=True)], None)] * 3
    model = SimpleNamespace(entry_needs=lambda: needs, rt=SimpleNamespace(dtype=torch.bfloat16, device="cuda:0"))
    free = 1_000_003
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda device=None: (free, free))
    for cache_dtype, kv_dtype in ((None, None), ("float8_e4m3", torch.float8_e4m3fn)):
        n = pages_for(model, page, 1 << 20, 1 << 20, 0.5, cache_dtype=cache_dtype)

        def size(pages):
            m = CacheManager(needs, pages, page, 1, torch.bfloat16, "cpu", 1 << 20, kv_dtype=kv_dtype)
            return sum(t.numel() * t.element_size() for g in m.copied_tensors() for t in g)
        assert size(n) <= free * 0.5 < size(n + 1)


@pytest.mark.parametrize("operation", [0, 1])
@pytest.mark.parametrize("page,hd", [(1 << 30, 8), (1 << 25, 64), ((1 << 30) + 16, 64), ((1 << 31) - 16, 8), (1 << 28, 8)])
def test_pages_whose_rows_pass_32_bits_are_refused(operation, page, hd):
    """A page of a head with 2^31 entries or more, before anything is launched (or counted towards)."""
    from gibbs_b200.ops.library import library
    lib = library("kv8")
    lib.gb_kv8_run.argtypes, lib.gb_kv8_run.restype = [ctypes.c_char_p], ctypes.c_int
    lib.gb_last_error.restype = ctypes.c_char_p
    heads, kv_heads, bf16 = 4, 2, 1
    if operation == 0:
        operands = [0, 8 * hd, bf16, 0, 0, 0, 0, 0, 0, 16, 16, 16, 16, 1, page, heads, kv_heads, hd, 0, 1]
    else:
        operands = [0, 4 * hd, bf16, 0, 4 * hd, 16, 16, 16, 16, 1, page, heads, kv_heads, hd, 0, 1, 0, 0, 0, 0]
    words = struct.pack("=18qd20q", operation, 0, 0, 1, 1, 0, 1, 1, 1, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0.125, *operands)
    assert lib.gb_kv8_run(words) < 0
    assert b"pages of" in lib.gb_last_error()
