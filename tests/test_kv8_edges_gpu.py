"""The 8-bit paged cache where its kernels meet what is not theirs: pages of other requests, the way from kernel to kernel, the
values of an argument at the ends of its range.  One way through every kernel each."""
import math
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
@pytest.mark.parametrize("way", WAYS)
def test_scales_below_zero_and_zero(way):
    """softmax(-s q K^T) V is that of -q under s, to the bit; under 0 every visible key has the same weight."""
    from gibbs_b200.ops import kv8
    dtype, heads, kv_heads, hd, page, portions = WAYS[way]
    behind = [(37 * i) % 90 for i in range(len(portions))]
    gen = torch.Generator().manual_seed(2)
    n_pages, bt = tables(portions, behind, page, random.Random(1))
    pages = make_pages(n_pages, kv_heads, page, hd, gen)
    q = torch.randn(sum(portions), heads * hd, generator=gen).to(dtype).to(DEV)
    call = lambda x, scale: kv8.paged_attention(x, heads, kv_heads, hd, pages, bt.to(DEV), scale, 0, torch.empty_like(q),  # noqa: E731
                                                step_of(portions, behind))
    assert torch.equal(call(q, -0.3), call(-q, 0.3)) and not torch.equal(call(q, -0.3), call(q, 0.3))
    got = call(q, 0.0).double().cpu().view(-1, kv_heads, heads // kv_heads, hd)
    values, row = pages.dequantized()[1].double().cpu(), 0
    for r, (p, b) in enumerate(zip(portions, behind)):
        n = b + p
        ids = bt[r, :-(-n // page)].long()
        for h in range(kv_heads):
            v = values[ids, h].reshape(-1, hd)[:n]
            upto = torch.arange(b + 1, n + 1).double()[:, None]
            want, weight = v.cumsum(0)[b:] / upto, v.abs().cumsum(0)[b:] / upto
            # 32-bit sums over n keys (2^-23 of their magnitudes each) and a quotient; in 16 bits a weight's rounding (2^-11 of it),
            # 2^-37 * 448 * (keys) * (the largest page scale over the keys) where a weight is that small, and the output's own (2^-8)
            tol = (n + 64) * 2.0 ** -23 * weight
            if dtype == torch.bfloat16:
                most = (pages.v_scales[ids.to(DEV), h].abs().max().item())
                tol = tol + 2.0 ** -11 * weight + 2.0 ** -37 * 448 * most + 2.0 ** -8 * want.abs()
            assert bool(((got[row:row + p, h] - want[:, None]).abs() <= tol[:, None]).all())
        row += p


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf, 1e39])
def test_scales_that_are_not_finite_are_refused(scale):
    from gibbs_b200.ops import KernelError, kv8
    for way in ("8 rows, 64", "256 rows, 64", "32 bits"):
        dtype, heads, kv_heads, hd, page, portions = WAYS[way]
        n_pages, bt = tables(portions, [0] * len(portions), page, random.Random(1))
        pages = make_pages(n_pages, kv_heads, page, hd, torch.Generator().manual_seed(2))
        q = torch.zeros(sum(portions), heads * hd, dtype=dtype, device=DEV)
        with pytest.raises(KernelError, match="scale"):
            kv8.paged_attention(q, heads, kv_heads, hd, pages, bt.to(DEV), scale, 0, torch.empty_like(q), step_of(portions, [0] * len(portions)))


@pytest.mark.parametrize("way", WAYS)
def test_store_and_attention_one_right_behind_the_other(way):
    """A step's store and attention launched without a pause, over other rows every time: each sees what the kernel in front wrote."""
    from gibbs_b200.ops import kv8
    dtype, heads, kv_heads, hd, page, portions = WAYS[way]
    behind = [(37 * i) % 90 for i in range(len(portions))]
    gen = torch.Generator().manual_seed(3)
    n_pages, bt = tables(portions, behind, page, random.Random(1))
    clean = make_pages(n_pages, kv_heads, page, hd, gen)
    rows = [torch.randn(sum(portions), (heads + 2 * kv_heads) * hd, generator=gen).to(dtype).to(DEV) for _ in range(8)]
    bt, step = bt.to(DEV), step_of(portions, behind)

    def run(pause):
        pages = kv8.Pages(*(t.clone() for t in clean.tensors()))
        outs = []
        torch.cuda.synchronize()
        for x in rows:
            q, out = (torch.empty(sum(portions), heads * hd, dtype=dtype, device=DEV) for _ in range(2))
            for _ in range(2):                                     # (the second over the first's pages, which lets the host run ahead)
                kv8.qk_norm_rope_store(x, q, heads, kv_heads, hd, None, None, 1e-5, None, 0, False, step, bt, pages)
                pause()
                kv8.paged_attention(q, heads, kv_heads, hd, pages, bt, hd ** -0.5, 0, out, step)
                pause()
            outs.append(out)
        return outs

    want = run(torch.cuda.synchronize)
    for _ in range(5):
        for a, b in zip(run(lambda: None), want):
            assert torch.equal(a, b)
    assert int(step.status.item()) == 0


def test_a_launch_without_work_ends_behind_the_kernel_in_front():
    """Requests without tokens (a padded step's): nothing is read or written, and what comes next still waits for what came before."""
    from gibbs_b200.ops import kv8
    gen = torch.Generator().manual_seed(4)
    for way in WAYS:
        dtype, heads, kv_heads, hd, page, portions = WAYS[way]
        n_pages, bt = tables(portions, [40] * len(portions), page, random.Random(1))
        pages, bt = make_pages(n_pages, kv_heads, page, hd, gen), bt.to(DEV)
        before = [bits(t).clone() for t in pages.tensors()]
        step, none = (step_of(portions, [40] * len(portions)) for _ in range(2))
        none.q_len = torch.zeros_like(none.q_len)
        n = sum(portions)
        x = torch.randn(n, (heads + 2 * kv_heads) * hd, generator=gen).to(dtype).to(DEV)
        q, out = (torch.full((n, heads * hd), 7.0, dtype=dtype, device=DEV) for _ in range(2))
        kv8.qk_norm_rope_store(x, q, heads, kv_heads, hd, None, None, 1e-5, None, 0, False, none, bt, pages)
        kv8.paged_attention(q, heads, kv_heads, hd, pages, bt, hd ** -0.5, 0, out, none)
        assert bool((q == 7.0).all()) and bool((out == 7.0).all())
        assert all(torch.equal(bits(a), b) for a, b in zip(pages.tensors(), before))
        kv8.qk_norm_rope_store(x, q, heads, kv_heads, hd, None, None, 1e-5, None, 0, False, step, bt, pages)
        kv8.paged_attention(torch.zeros_like(q), heads, kv_heads, hd, pages, bt, hd ** -0.5, 0, out, none)
        got = kv8.paged_attention(q, heads, kv_heads, hd, pages, bt, hd ** -0.5, 0, torch.empty_like(q), step)
        torch.cuda.synchronize()
        assert torch.equal(got, kv8.paged_attention(q, heads, kv_heads, hd, pages, bt, hd ** -0.5, 0, out, step))
        assert int(step.status.item()) == 0


@pytest.mark.parametrize("way", ["256 rows, 64", "256 rows, 128", "256 rows beside 8"])
def test_products_store_and_attention_on_two_streams_without_a_pause(way):
    """Layers' worth of (product, store, attention, product), whose kernels share the SMs' tensor memory, in one stream and in two at
    once: every run ends and gives the same bits."""
    from gibbs_b200 import ops
    from gibbs_b200.ops import kv8
    dtype, heads, kv_heads, hd, page, portions = WAYS[way]
    n, behind, wide = sum(portions), [(37 * i) % 90 for i in range(len(portions))], (heads + 2 * kv_heads) * hd
    gen = torch.Generator().manual_seed(5)
    n_pages, bt = tables(portions, behind, page, random.Random(1))
    bt, step = bt.to(DEV), step_of(portions, behind)
    w_in, w_out = ((torch.randn(a, b, generator=gen) * b ** -0.5).to(dtype).to(DEV) for a, b in ((wide, 512), (512, heads * hd)))
    x0, clean = torch.randn(n, 512, generator=gen).to(dtype).to(DEV), make_pages(n_pages, kv_heads, page, hd, gen)

    def layers():
        pages, x = kv8.Pages(*(t.clone() for t in clean.tensors())), x0
        for _ in range(12):
            rows, q, out, y = (torch.empty(n, c, dtype=dtype, device=DEV) for c in (wide, heads * hd, heads * hd, 512))
            ops.linear(x, w_in, None, rows)
            kv8.qk_norm_rope_store(rows, q, heads, kv_heads, hd, None, None, 1e-5, None, 0, False, step, bt, pages)
            kv8.paged_attention(q, heads, kv_heads, hd, pages, bt, hd ** -0.5, 0, out, step)
            x = ops.linear(out, w_out, None, y)
        return x

    want = layers()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(4):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append(layers())
        torch.cuda.synchronize()
        assert all(torch.equal(g, want) for g in got) and not bool(want.isnan().any())
    assert int(step.status.item()) == 0


@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("portions", [[20, 20, 20], [13, 60, 60], [12, 60, 60], [1, 60, 60], [60, 0, 60], [13, 14, 13]])
def test_steps_at_the_border_of_what_one_launch_takes(portions, hd, page):
    """Groups of four heads: 13 tokens are more than 48 rows and 12 are not.  Each request gets what it gets alone, to a bfloat16's last
    place of what its sums go over; rows behind the tokens are left, also where a step counts more tokens than its requests bring."""
    from gibbs_b200.ops import kv8
    heads, kv_heads, behind = 32, 8, [70, 300, 5]
    gen = torch.Generator().manual_seed(6)
    n_pages, bt = tables(portions, behind, page, random.Random(1))
    pages, bt = make_pages(n_pages, kv_heads, page, hd, gen), bt.to(DEV)
    n = sum(portions)
    q = torch.randn(n + 9, heads * hd, generator=gen).to(torch.bfloat16).to(DEV)
    for more in (0, 9):
        step = step_of(portions, behind)
        step.n_tokens += more
        out = kv8.paged_attention(q, heads, kv_heads, hd, pages, bt, hd ** -0.5, 0, torch.full_like(q, 7.0), step)
        assert bool((out[n:] == 7.0).all()) and int(step.status.item()) == 0
        at = 0
        for r, (p, b) in enumerate(zip(portions, behind)):
            if not p:
                continue
            alone = kv8.paged_attention(q[at:at + p], heads, kv_heads, hd, pages, bt[r:r + 1], hd ** -0.5, 0, torch.empty_like(q[at:at + p]), step_of([p], [b]))
            # (weights in f16 under another running maximum: 2^-11 of them each, twice; and the output's rounding, twice)
            size = pages.dequantized()[1][bt[r, :-(-(p + b) // page)].long()].abs().amax().item()
            assert bool(((out[at:at + p].float() - alone.float()).abs() <= 2 * 2.0 ** -11 * size + 2 * 2.0 ** -8 * alone.float().abs()).all())
            at += p
