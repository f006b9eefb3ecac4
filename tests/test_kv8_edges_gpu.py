"""The 8-bit paged cache where its kernels meet what is not theirs: pages of other requests, the way from kernel to kernel, the
values of an argument at the ends of its range.  One way through every kernel each."""
import random

import pytest
import torch

from test_kv8_gpu import DEV, bits, make_pages, step_of, tables

pytestmark = pytest.mark.gpu

# dtype, heads, kv_heads, hd, page, tokens of a request, requests: tiles of 8 rows by many and by few warps, of 16 rows, of 256 rows
# (alone, beside single tokens), and the kernels of any type, head size and page size
WAYS = {
    "8 rows, 64": (torch.bfloat16, 32, 8, 64, 16, [1] * 6),
    "8 rows, 128": (torch.bfloat16, 16, 4, 128, 64, [1] * 6),
    "8 rows, many": (torch.bfloat16, 32, 8, 64, 16, [1] * 40),
    "16 rows, 64": (torch.bfloat16, 32, 8, 64, 16, [3] * 36),
    "16 rows, 128": (torch.bfloat16, 32, 8, 128, 32, [3] * 36),
    "256 rows, 64": (torch.bfloat16, 24, 8, 64, 16, [200]),
    "256 rows, 128": (torch.bfloat16, 16, 4, 128, 64, [150, 70]),
    "256 rows beside 8": (torch.bfloat16, 24, 8, 64, 16, [200, 1, 1, 37, 1, 1]),
    "32 bits": (torch.float32, 24, 8, 64, 16, [1, 1, 3, 1, 1, 9]),
    "any, 16 bits": (torch.bfloat16, 4, 2, 96, 16, [1, 1, 3, 1, 1, 9]),
    "any, 32 bits": (torch.float32, 5, 1, 24, 5, [1, 1, 3, 1, 1, 9]),
}


@pytest.mark.parametrize("window", [40, 57])
@pytest.mark.parametrize("way", WAYS)
def test_nan_in_pages_that_a_request_does_not_hold(way, window):
    """Every page that no table names is NaN throughout, the pool's first among them; windows begin in every quarter of a
    chunk of keys.  What a request gets is what it gets beside clean pages, to the bit."""
    from gibbs_b200.ops import kv8
    dtype, heads, kv_heads, hd, page, portions = WAYS[way]
    firsts = [0, 15, 16, 31, 48, 177]                              # a request's first token sees keys from here on
    behind = [firsts[i % len(firsts)] + window - 1 for i in range(len(portions))]
    gen = torch.Generator().manual_seed(1)
    n_pages, bt = tables(portions, behind, page, random.Random(1), spare=2, holes=[(b - window + 1) // page for b in behind])
    bt[bt >= 0] += 1                                               # (page 0 is nobody's)
    n_pages += 1
    pages = make_pages(n_pages, kv_heads, page, hd, gen)
    q = torch.randn(sum(portions), heads * hd, generator=gen).to(dtype).to(DEV)
    step = step_of(portions, behind)
    call = lambda: kv8.paged_attention(q, heads, kv_heads, hd, pages, bt.to(DEV), hd ** -0.5, window, torch.empty_like(q), step)  # noqa: E731
    want = call()
    foreign = sorted(set(range(n_pages)) - set(bt.flatten().tolist()))
    assert 0 in foreign and len(foreign) >= 3
    for sign in (1.0, -1.0):
        for t, s in ((pages.k, pages.k_scales), (pages.v, pages.v_scales)):
            bits(t)[foreign] = 0x7f
            s[foreign] = sign * s[foreign].abs()
        got = call()
        assert int(step.status.item()) == 0 and not bool(got.isnan().any())
        assert torch.equal(got, want)
