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
