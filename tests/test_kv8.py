"""What the 8-bit cache and the row copies refuse, as far as it needs no GPU."""
import ctypes
import math
import struct

import pytest
import torch

import plain_kv8 as plain

F8 = torch.float8_e4m3fn


def test_pages_are_checked():
    from gibbs_b200.ops import KernelError, kv8
    k = torch.zeros(3, 2, 16, 64).to(F8)
    s = torch.ones(3, 2)
    p = kv8.Pages(k, k.clone(), s, s.clone())
    assert (p.n_pages, p.kv_heads, p.page_size, p.head_dim) == (3, 2, 16, 64)
    for bad in ((k.float(), k, s, s), (k, k[:2], s, s), (k, k, s[:, :1], s), (k, k, s, s.double()), (k[0], k[0], s, s),
                (k.transpose(1, 2), k.transpose(1, 2), s, s), (k[..., :60].contiguous(), k[..., :60].contiguous(), s, s)):
        with pytest.raises(KernelError):
            kv8.Pages(*bad)
    with pytest.raises(KernelError):
        kv8.check_head_dim(264)
    k2, v2 = p.dequantized()
    assert k2.shape == k.shape and k2.dtype == torch.float32


def test_operations_need_cuda_tensors():
    from gibbs_b200.ops import KernelError, RowCopies, kv8
    k = torch.zeros(3, 2, 16, 64).to(F8)
    p = kv8.Pages(k, k.clone(), torch.ones(3, 2), torch.ones(3, 2))
    x = torch.zeros(1, 8 * 64)
    with pytest.raises(KernelError):
        kv8.qk_norm_rope_store(x, x[:, :256], 4, 2, 64, None, None, 0.0, None, 0, False, None, x, p)
    with pytest.raises(KernelError):
        kv8.paged_attention(x[:, :256], 4, 2, 64, p, x, 1.0, 0, x[:, :256], None)
    with pytest.raises(KernelError):
        RowCopies([[x]])


@pytest.mark.parametrize("pairs", [[(0, 10)], [(10, 0)], [(-1, 2)], [(3, 3)], [(0, 1), (2, 1)], [(0, 1), (1, 2)], [(1, 2), (0, 1)]])
def test_pairs_are_checked_before_anything_is_launched(pairs):
    """The check itself, in the library: rows outside the group, a destination twice, a destination that is a source."""
    from gibbs_b200.ops.library import library
    lib = library("kv8")
    n, flat = len(pairs), [v for p in pairs for v in p]
    arr = (ctypes.c_int * len(flat))(*flat)
    lib.gb_row_copies.argtypes, lib.gb_row_copies.restype = [ctypes.c_char_p], ctypes.c_int
    assert lib.gb_row_copies(struct.pack("=7q", 0, 0, 1, ctypes.addressof(arr), n, 1, 10)) < 0
    lib.gb_last_error.restype = ctypes.c_char_p
    assert b"row copies" in lib.gb_last_error()


def test_scales_of_the_oracle():
    assert plain.scale_for(448.0) == 1.0 and plain.scale_for(448.1) == 2.0 and plain.scale_for(0.0) == 2.0 ** -64
    assert plain.scale_for(224.0) == 0.5 and plain.scale_for(1.0) == 2.0 ** -8 and plain.scale_for(448 * 2.0 ** 50) == 2.0 ** 50
    x = torch.tensor([448.0, 0.0625, 2.0 ** -10, 2.0 ** -9 * 1.5, 17.0, math.nan], dtype=torch.float64)
    y = plain.to_e4m3(x)
    assert y[:5].tolist() == [448.0, 0.0625, 0.0, 2.0 ** -8, 16.0] and math.isnan(float(y[5]))
