"""The 8-bit paged cache against its definition in 64 bits: storing, attention of single tokens and of portions, row copies."""
import math
import random
from types import SimpleNamespace

import pytest
import torch

import plain_kv8 as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F8 = torch.float8_e4m3fn
EPS = 1e-5


def step_of(portions, behind, dev=DEV):
    from gibbs_b200 import ops
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)                                     # noqa: E731
    starts = [sum(portions[:r]) for r in range(len(portions))]
    return SimpleNamespace(n_tokens=sum(portions), n_requests=len(portions), q_start=i32(starts), q_len=i32(portions),
                           start_pos=i32(behind), max_q_len=max(portions), max_ctx_len=max(p + b for p, b in zip(portions, behind)),
                           status=ops.device_status(torch.device(dev)))


def tables(portions, behind, page, rng, spare=3, holes=()):
    """Random distinct pages for every request; the pages of ``holes`` (window passed) are -1."""
    blocks = [-(-(p + b) // page) for p, b in zip(portions, behind)]
    n = sum(blocks) + spare
    ids = list(range(n))
    rng.shuffle(ids)
    width = max(max(blocks), 1)
    out, at = [], 0
    for r, b in enumerate(blocks):
        row = ids[at:at + b] + [-1] * (width - b)
        at += b
        for j in range(holes[r] if holes else 0):
            row[j] = -1
        out.append(row)
    return n, torch.tensor(out, dtype=torch.int32)


def make_pages(n_pages, kv_heads, page, hd, gen, size=1.0):
    """Pages that hold something everywhere: random numbers under random scales."""
    from gibbs_b200.ops import kv8
    t = []
    for _ in range(2):
        t.append((torch.randn(n_pages, kv_heads, page, hd, generator=gen) * 100).clamp(-448, 448).to(F8).to(DEV))
    for _ in range(2):
        t.append((size * torch.exp2(torch.randint(-9, -6, (n_pages, kv_heads), generator=gen).float())).to(DEV))
    return kv8.Pages(t[0], t[1], t[2], t[3])


def bits(t):
    return t.view(torch.uint8) if t.dtype == F8 else t


STORES = [
    # dtype, heads, kv_heads, hd, page, rotation (rotary_dim, adjacent), norm, portions, behind
    ("bf16", 32, 8, 64, 16, (64, False), True, [1], [0]),
    ("bf16", 32, 8, 64, 16, (64, False), True, [1] * 9, [0, 1, 15, 16, 17, 31, 100, 4095, 30000]),
    ("bf16", 4, 2, 64, 16, (64, False), True, [7, 1, 40, 16, 1], [0, 3, 9, 16, 15]),
    ("bf16", 4, 4, 128, 64, (128, False), True, [200, 1, 63], [0, 64, 60]),
    ("bf16", 6, 2, 128, 128, (128, False), False, [150, 3], [100, 0]),
    ("bf16", 3, 1, 64, 8, (64, False), True, [33, 1, 1], [5, 7, 8]),
    ("bf16", 4, 2, 16, 16, (16, False), True, [20, 1], [10, 2]),
    ("bf16", 4, 2, 64, 16, (32, False), True, [20, 1], [10, 2]),
    ("bf16", 4, 2, 64, 16, (64, True), True, [20, 1], [10, 2]),
    ("bf16", 2, 1, 256, 16, (256, False), True, [18], [15]),
    ("bf16", 2, 1, 96, 5, (96, False), True, [18, 1], [3, 4]),
    ("bf16", 4, 2, 64, 32, None, False, [50, 1, 1], [31, 31, 32]),
    ("f32", 32, 8, 64, 16, (64, False), True, [1] * 5, [0, 1, 15, 16, 30000]),
    ("f32", 4, 2, 64, 16, (64, False), True, [7, 1, 40, 16, 1], [0, 3, 9, 16, 15]),
    ("f32", 4, 2, 128, 64, (128, False), True, [130, 1, 65], [0, 64, 63]),
    ("f32", 3, 1, 24, 16, (8, True), False, [5, 20], [14, 0]),
]


def store_case(dtype, heads, kv_heads, hd, page, rotation, norm, portions, behind, seed=0, spoil=None, pad=0, wide=0, size=1.0):
    """Runs a store on the GPU and in 64 bits; returns what both left."""
    from gibbs_b200 import ops
    from gibbs_b200.ops import kv8
    gen, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    n, slots = sum(portions), heads + 2 * kv_heads
    n_pages, bt = tables(portions, behind, page, rng)
    pages = make_pages(n_pages, kv_heads, page, hd, gen)
    x = (torch.randn(n + pad, slots * hd + wide, generator=gen) * torch.exp(torch.randn(n + pad, 1, generator=gen)) * size).to(dt)
    if spoil is not None:
        spoil(x)
    gains = [1 + 0.2 * torch.randn(hd, generator=gen) if norm else None for _ in range(2)]
    freq = None
    if rotation is not None:
        freq = 10000.0 ** (-torch.arange(0, rotation[0], 2).double() / rotation[0])
        table = torch.cat([freq.float(), torch.tensor([1.25])])
        freq = table[:-1]
    before = [bits(t).clone() for t in pages.tensors()]
    step = step_of(portions, behind)
    q_out = torch.full((n + pad, heads * hd), 7.0, dtype=dt, device=DEV)
    dev = lambda t: None if t is None else t.to(DEV)                                                  # noqa: E731
    kv8.qk_norm_rope_store(x.to(DEV)[:, :slots * hd] if wide else x.to(DEV), q_out, heads, kv_heads, hd, dev(gains[0]), dev(gains[1]),
                           EPS, None if rotation is None else table.to(DEV), 0 if rotation is None else rotation[0],
                           False if rotation is None else rotation[1], step, bt.to(DEV), pages)
    assert int(step.status.item()) == 0
    # in 64 bits
    pos = torch.cat([torch.arange(b, b + p) for p, b in zip(portions, behind)])
    y = x[:n, :slots * hd].double().view(n, slots, hd)
    rot = (freq, 1.25, 0 if rotation is None else rotation[0], False if rotation is None else rotation[1], pos)
    q = plain.rotated(y[:, :heads], gains[0], EPS, *rot)
    k = plain.rotated(y[:, heads:heads + kv_heads], gains[1], EPS, *rot)
    v = y[:, heads + kv_heads:]
    want = []
    for codes, scales, rows in ((before[0].view(F8), before[2], k), (before[1].view(F8), before[3], v)):
        pp = plain.PlainPages(codes, scales)
        row = 0
        for r, (p, b) in enumerate(zip(portions, behind)):
            at = b
            while at < b + p:
                m = min(page - at % page, b + p - at)
                pp.store(int(bt[r, at // page]), at % page, rows[row:row + m])
                at, row = at + m, row + m
        want.append(pp)
    return SimpleNamespace(pages=pages, before=before, q_out=q_out.cpu(), q=q.reshape(n, -1), want=want, n=n, ops=ops, dt=dt,
                           bt=bt, step=step, y=y, rows=(k, v))


# 32-bit sums of up to 256 squares, a reciprocal root, a rotation: within 2^-18 of the head's largest magnitude
F32_SLACK = 2.0 ** -18


def check_store(c, page):
    n = c.n
    half_step = torch.finfo(c.dt).eps / 2
    big = c.q.abs().amax()
    head = c.q.view(n, -1)
    err = (c.q_out[:n].double() - head).abs()
    assert bool((err <= half_step * head.abs() + F32_SLACK * (head.abs().amax(-1, keepdim=True) + 1e-30)).all()), (err.max(), big)
    assert bool((c.q_out[n:] == 7.0).all())
    for codes, scales, want, old in ((c.pages.k, c.pages.k_scales, c.want[0], (c.before[0], c.before[2])),
                                     (c.pages.v, c.pages.v_scales, c.want[1], (c.before[1], c.before[3]))):
        got, s = codes.cpu().float().double(), scales.cpu().double()
        touched = want.written.any(1)
        # pages that no token went to are as they were, and so is every row that is neither new nor re-rounded
        assert torch.equal(bits(codes).cpu()[~touched], old[0].cpu()[~touched])
        assert torch.equal(scales.cpu()[~touched], old[1].cpu()[~touched])
        keep = want.slack == 0
        keep &= ~want.written[:, None, :, None]
        assert torch.equal(bits(codes).cpu()[keep], old[0].cpu()[keep])
        # scales: equal, but where the largest magnitude lies within 32-bit error of 448 2^e
        differ = s != want.s
        for i, h in differ.nonzero().tolist():
            top = float(want.ideal[i, h][want.written[i]].nan_to_num().abs().max())
            near = min(abs(top / (448 * 2.0 ** e) - 1) for e in range(-64, 51))
            assert near < F32_SLACK and 0.5 <= float(s[i, h].abs() / want.s[i, h].abs()) <= 2, (i, h, s[i, h], want.s[i, h])
        value = got * s.abs()[:, :, None, None]
        ideal = want.ideal[touched]
        v, sc = value[touched], s.abs()[touched][:, :, None, None]
        rows = (want.written | (want.slack > 0).any(-1).any(1))[touched][:, None, :, None].expand_as(v)
        nan = ideal.isnan()
        assert torch.equal(v.isnan() & rows, nan & rows)
        mag = ideal.nan_to_num().abs()
        tol = torch.maximum(2.0 ** -4 * mag, 2.0 ** -10 * sc) + want.slack[touched] \
            + F32_SLACK * mag.amax(-1, keepdim=True) * (1 + 2.0 ** -4)
        # (a row that was re-rounded lies on the grid of its first rounding, which `ideal` holds)
        bad = ((v - ideal).abs() > tol) & rows & ~nan
        assert not bool(bad.any()), (int(bad.sum()), (v - ideal).abs()[bad][:5], tol[bad][:5])


@pytest.mark.parametrize("case", STORES, ids=[f"{i}-{c[0]}-{c[3]}-{c[4]}" for i, c in enumerate(STORES)])
def test_store_against_its_definition(case):
    check_store(store_case(*case), case[4])


def test_store_reads_strided_rows_and_leaves_rows_behind_the_last_token():
    for case in (STORES[2], STORES[13]):
        check_store(store_case(*case, pad=5, wide=64), case[4])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64), (40, 16)])
def test_a_page_filled_token_by_token_with_growing_values(dtype, hd, page):
    """Each token is larger than the one before: the scale grows and every row is rounded again.  Codes and scales equal the
    definition's, applied in the same order (v is taken as it is: nothing but the roundings can differ)."""
    from gibbs_b200.ops import kv8
    gen = torch.Generator().manual_seed(3)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    kv_heads = 2
    pages = make_pages(3, kv_heads, page, hd, gen)
    bt = torch.tensor([[2, 0]], dtype=torch.int32, device=DEV)
    want = plain.PlainPages(pages.v, pages.v_scales)
    for pos in range(page + 3):
        x = torch.randn(1, (1 + 2 * 1) * 0 + 4 * hd + 2 * kv_heads * hd, generator=gen) * 1.3 ** (pos if pos < page else 0) * 1e-3
        x = x.to(dt)
        q_out = torch.empty(1, 4 * hd, dtype=dt, device=DEV)
        kv8.qk_norm_rope_store(x.to(DEV), q_out, 4, kv_heads, hd, None, None, EPS, None, 0, False, step_of([1], [pos]), bt, pages)
        want.store(int(bt[0, pos // page]), pos % page, x[:, 4 * hd + kv_heads * hd:].view(1, kv_heads, hd).double())
    assert torch.equal(pages.v_scales.cpu().double(), want.s)
    assert torch.equal(pages.v.cpu().float().double(), want.n)


@pytest.mark.parametrize("scale", [0.0, 1e-30, 2.0 ** -64, 448 * 2.0 ** 50, 1e30])
def test_the_smallest_and_largest_magnitudes(scale):
    """Rows of zeros, of values under the smallest scale, at the largest magnitude, and above it (NaN)."""
    def fill(x):
        x.fill_(scale)
        x[:, ::3] *= -1
    c = store_case("f32", 4, 2, 64, 16, None, False, [20, 1], [3, 15], spoil=fill)
    check_store(c, 16)
    if scale == 0.0:
        assert bool((c.pages.v_scales.cpu()[c.want[1].written.any(1)] > 0).all())


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("portions,behind", [([40, 1], [0, 5]), ([1, 1, 1], [5, 16, 31])])
def test_values_that_are_not_finite_are_stored_as_nan_and_mark_their_page(value, portions, behind):
    for dtype in ("bf16", "f32"):
        def spoil(x):
            x[0, 4 * 64 + 2 * 64 + 5] = value               # v of token 0, head 0
            x[-1, 4 * 64 + 64 + 9] = value                  # k of the last token, head 1
        c = store_case(dtype, 4, 2, 64, 16, None, False, portions, behind, spoil=spoil)
        check_store(c, 16)
        assert bool((c.pages.v_scales < 0).any()) and bool((c.pages.k_scales < 0).any())


def test_a_page_begins_anew_with_its_first_row():
    """Whatever an earlier owner left (a larger scale, the NaN mark, NaN rows) is gone when row 0 is written."""
    from gibbs_b200.ops import kv8
    for portion in (1, 5):
        pages = kv8.Pages(torch.full((2, 1, 16, 64), math.nan).to(F8).to(DEV), torch.full((2, 1, 16, 64), math.nan).to(F8).to(DEV),
                          torch.full((2, 1), -1024.0, device=DEV), torch.full((2, 1), -1024.0, device=DEV))
        x = torch.ones(portion, 3 * 64, dtype=torch.bfloat16, device=DEV)
        q = torch.empty(portion, 64, dtype=torch.bfloat16, device=DEV)
        bt = torch.tensor([[1]], dtype=torch.int32, device=DEV)
        kv8.qk_norm_rope_store(x, q, 1, 1, 64, None, None, EPS, None, 0, False, step_of([portion], [0]), bt, pages)
        assert float(pages.v_scales[1, 0]) == 2.0 ** -8 and float(pages.k_scales[1, 0]) == 2.0 ** -8
        k, v = pages.dequantized()
        assert bool((k[1, 0, :portion] == 1).all()) and bool((v[1, 0, :portion] == 1).all())
        assert bool(v[1, 0, portion:].isnan().all()) and bool(v[0].isnan().all())


@pytest.mark.parametrize("m", [1, 5, 40])
def test_store_of_partial_tiles_equals_the_store_of_their_sum(m):
    from gibbs_b200 import ops
    from gibbs_b200.ops import kv8
    gen = torch.Generator().manual_seed(m)
    heads, kv_heads, hd, page = 8, 2, 64, 16
    cols = (heads + 2 * kv_heads) * hd
    ws = torch.randn(3, m, cols, generator=gen).to(DEV)
    bias = torch.randn(cols, generator=gen).to(DEV)
    total = (((ws[0] + ws[1]) + ws[2]) + bias).to(torch.bfloat16)
    gain = (1 + 0.1 * torch.randn(hd, generator=gen)).to(DEV)
    table = torch.cat([10000.0 ** (-torch.arange(0, hd, 2).float() / hd), torch.ones(1)]).to(DEV)
    left = []
    for portions, behind in ([m], [3]), ([1] * m, list(range(m))):
        n_pages, bt = tables(portions, behind, page, random.Random(0))
        for rows in (total, ops.Partials(ws, bias, torch.bfloat16)):
            pages = make_pages(n_pages, kv_heads, page, hd, torch.Generator().manual_seed(1))
            q = torch.empty(m, heads * hd, dtype=torch.bfloat16, device=DEV)
            kv8.qk_norm_rope_store(rows, q, heads, kv_heads, hd, gain, gain, EPS, table, hd, False, step_of(portions, behind),
                                   bt.to(DEV), pages)
            left.append([q] + [bits(t) for t in pages.tensors()])
        for a, b in zip(left[-1], left[-2]):
            assert torch.equal(a, b)


def test_queries_alone_for_a_layer_that_reads_anothers_cache():
    from gibbs_b200.ops import kv8
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(7, 4 * 64, generator=gen).to(torch.bfloat16)
    q = torch.empty(7, 4 * 64, dtype=torch.bfloat16, device=DEV)
    table = torch.cat([10000.0 ** (-torch.arange(0, 64, 2).float() / 64), torch.ones(1)])
    kv8.qk_norm_rope_store(x.to(DEV), q, 4, 2, 64, None, None, EPS, table.to(DEV), 64, False, step_of([7], [11]),
                           torch.zeros(1, 2, dtype=torch.int32, device=DEV), None)
    want = plain.rotated(x.view(7, 4, 64), None, EPS, table[:-1], 1.0, 64, False, torch.arange(11, 18)).reshape(7, -1)
    assert bool(((q.cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + F32_SLACK * want.abs().amax()).all())


# ---------------------------------------------------------------------------------------------------
ATTENTIONS = [
    # dtype, heads, kv_heads, hd, page, window, portions, behind
    ("bf16", 32, 8, 64, 16, 0, [1], [0]),
    ("bf16", 32, 8, 64, 16, 0, [1] * 8, [0, 1, 7, 8, 15, 16, 31, 32]),
    ("bf16", 32, 8, 64, 16, 0, [1] * 5, [63, 64, 500, 1999, 4100]),
    ("bf16", 32, 8, 64, 16, 100, [1] * 5, [63, 99, 100, 101, 1999]),
    ("bf16", 16, 4, 128, 64, 0, [1] * 4, [0, 63, 64, 3000]),
    ("bf16", 24, 8, 64, 16, 0, [3, 1, 5, 2], [10, 700, 0, 31]),
    ("bf16", 24, 8, 64, 16, 0, [200, 1, 37, 130], [150, 300, 0, 14]),
    ("bf16", 32, 8, 64, 16, 70, [200, 1, 37, 130], [150, 300, 0, 14]),
    ("bf16", 4, 4, 64, 32, 0, [300, 1], [0, 256]),
    ("bf16", 8, 1, 64, 64, 0, [90, 33], [500, 0]),
    ("bf16", 16, 1, 128, 128, 0, [40, 1], [200, 127]),
    ("bf16", 16, 4, 128, 16, 0, [260, 20], [0, 100]),
    ("bf16", 40, 8, 64, 8, 0, [100, 1], [30, 9]),
    ("bf16", 14, 2, 64, 16, 0, [64, 1], [1, 500]),
    ("bf16", 32, 1, 64, 16, 0, [9, 1], [100, 15]),
    ("bf16", 4, 2, 16, 16, 0, [40, 1], [3, 70]),
    ("bf16", 4, 2, 32, 8, 0, [40, 1, 1], [3, 70, 0]),
    ("bf16", 4, 2, 96, 16, 0, [40, 1, 1], [3, 70, 0]),
    ("bf16", 4, 2, 256, 16, 0, [20, 1], [3, 70]),
    ("bf16", 4, 2, 64, 5, 0, [20, 1], [3, 70]),
    ("bf16", 4, 2, 64, 24, 0, [40, 1], [3, 70]),
    ("f32", 32, 8, 64, 16, 0, [1] * 5, [0, 15, 16, 500, 2100]),
    ("f32", 24, 8, 64, 16, 50, [1, 40, 3], [300, 20, 0]),
    ("f32", 4, 2, 128, 64, 0, [70, 1], [0, 900]),
    ("f32", 5, 1, 24, 16, 0, [30, 1], [2, 40]),
]


def attention_case(dtype, heads, kv_heads, hd, page, window, portions, behind, seed=0, spoil=None, pad=0, sharp=1.0):
    from gibbs_b200.ops import kv8
    gen, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    n, group = sum(portions), heads // kv_heads
    holes = [max(0, b - window + 1) // page if window else 0 for b in behind]
    n_pages, bt = tables(portions, behind, page, rng, holes=holes)
    pages = make_pages(n_pages, kv_heads, page, hd, gen, size=1.5 ** 0)
    if spoil is not None:
        spoil(pages, bt)
    wide = torch.randn(n + pad, heads * hd + 32, generator=gen).to(dt) * sharp
    out = torch.full((n + pad, heads * hd), 7.0, dtype=dt, device=DEV)
    step = step_of(portions, behind)
    scale = hd ** -0.5
    kv8.paged_attention(wide.to(DEV)[:, :heads * hd], heads, kv_heads, hd, pages, bt.to(DEV), scale, window, out, step)
    assert int(step.status.item()) == 0
    keys, values = (t.double().cpu() for t in pages.dequantized())
    q = wide[:n, :heads * hd].double().view(n, kv_heads, group, hd)
    want, weight, spread, largest = (torch.zeros(n, kv_heads, group, hd, dtype=torch.float64) for _ in range(4))
    scales = pages.v_scales.abs().double().cpu()
    row = 0
    for r, (p, b) in enumerate(zip(portions, behind)):
        ids = bt[r, :-(-(p + b) // page)].long().clamp(min=0)
        for h in range(kv_heads):
            k, v = (t[ids, h].reshape(-1, hd) for t in (keys, values))
            s = slice(row, row + p)
            want[s, h], weight[s, h], spread[s, h], largest[s, h] = plain.attention(
                q[s, h], k, v, scale, window, torch.arange(b, b + p), scales[ids, h].repeat_interleave(page))
        row += p
    got = out.cpu()
    assert bool((got[n:] == 7.0).all())
    most = max(p + b for p, b in zip(portions, behind))
    # scores: hd products summed in 32 bits, each sum off by 2^-23 of the magnitudes it goes over (tensor cores cut off), so a
    # weight is off by twice hd * 2^-23 of the largest sum of magnitudes; sums over the keys likewise
    soft = 2 * (hd + 8) * 2.0 ** -23 * spread + (most + 64) * 2.0 ** -23
    tol = soft * weight + (2.0 ** -18 * weight)
    if dt == torch.bfloat16:
        tol = tol + 2.0 ** -8 * weight + 2.0 ** -8 * want.abs()          # weights in 16 bits, and the output's own rounding
        # Weights p_j s_j (s_j: the page's scale) are held in f16 as w = p_j s_j 2^12 / u, u the largest that the running maximum
        # has seen (or up to 2^3 below it), so u <= max_j p_j s_j.  An f16 of w is off by 2^-25 at most where it is subnormal:
        # an output by sum_j 2^-25 2^-12 u |n_j| <= 2^-37 * 448 * (number of keys) * max_j p_j s_j.
        tol = tol + 2.0 ** -37 * 448 * largest
    return got[:n].double().view(want.shape), want, tol


def check_attention(got, want, tol):
    assert torch.equal(got.isnan(), want.isnan())
    fine = ~want.isnan()
    bad = ((got - want).abs() > tol) & fine
    assert not bool(bad.any()), (int(bad.sum()), (got - want).abs()[bad][:5], tol[bad][:5], bad.nonzero()[:5])


@pytest.mark.parametrize("case", ATTENTIONS, ids=[f"{i}-{c[0]}-{c[1]}-{c[2]}-{c[3]}-{c[4]}" for i, c in enumerate(ATTENTIONS)])
def test_attention_against_its_definition(case):
    check_attention(*attention_case(*case, pad=3))


@pytest.mark.parametrize("case", [ATTENTIONS[i] for i in (2, 4, 5, 6, 11, 22)])
def test_attention_with_sharp_scores(case):
    """A few keys carry the weight: a lost key or a wrong edge shows."""
    check_attention(*attention_case(*case, sharp=4.0, seed=5))


@pytest.mark.parametrize("case", [ATTENTIONS[i] for i in (2, 4, 6, 7, 10, 11, 12, 15, 21, 22)])
def test_nan_stays_with_the_rows_that_see_it(case):
    """A NaN among the keys or values of one page, whose scale says so, reaches exactly the rows and columns that see it."""
    def spoil(pages, bt):
        page, r = case[4], len(case[7]) - 1
        end = case[6][r] + case[7][r]
        for j, (t, s) in ((end - 1, (pages.v, pages.v_scales)), (max(0, end - 12), (pages.v, pages.v_scales)),
                          (case[6][0] + case[7][0] - 2, (pages.k, pages.k_scales))):
            r_ = r if t is pages.v else 0
            if j < 0:
                continue
            i = int(bt[r_, j // page])
            if i < 0:
                continue
            bits(t)[i, 0, j % page, 3] = 0x7f
            s[i, 0] = -s[i, 0].abs()
    check_attention(*attention_case(*case, spoil=spoil))


@pytest.mark.parametrize("case", [ATTENTIONS[i] for i in (2, 4, 6, 11, 12, 15, 21)])
def test_pages_of_every_scale(case):
    """Scales far from one another, large ones (beyond 2^7) and numbers below 2^-6 of their scale among them."""
    def spoil(pages, bt):
        g = torch.Generator().manual_seed(9)
        pages.k_scales.mul_(torch.exp2(torch.randint(-3, 2, pages.k_scales.shape, generator=g).float()).to(DEV))
        pages.v_scales.copy_(torch.exp2(torch.randint(-30, 20, pages.v_scales.shape, generator=g).float()).to(DEV))
        small = torch.randint(0, 2, pages.k.shape, generator=g).to(DEV).bool()
        bits(pages.k)[small] = bits(pages.k)[small] & 0x87          # subnormal numbers
        bits(pages.v)[small] = bits(pages.v)[small] & 0x87
    check_attention(*attention_case(*case, spoil=spoil))


def test_stale_rows_behind_the_context_do_not_matter():
    """NaN and large numbers in rows that no token has written yet, in the page the context ends in."""
    for case in (ATTENTIONS[1], ATTENTIONS[6], ATTENTIONS[11], ATTENTIONS[21]):
        def spoil(pages, bt):
            for r, (p, b) in enumerate(zip(case[6], case[7])):
                end, page = p + b, case[4]
                if end % page:
                    i = int(bt[r, end // page])
                    for t in (pages.k, pages.v):
                        bits(t)[i, :, end % page:] = 0x7f
        # (the oracle must not see them either: rows past the context are hidden by its mask, but 0 * NaN is not)
        got, want, tol = attention_case(*case, spoil=spoil)
        check_attention(got, want, tol)


def test_padded_batch_requests_without_tokens_and_repeated_pages():
    from gibbs_b200.ops import kv8
    gen = torch.Generator().manual_seed(2)
    pages = make_pages(6, 2, 16, 64, gen)
    bt = torch.tensor([[0, 1, 2], [3, 3, 3], [0, 1, 2]], dtype=torch.int32, device=DEV)     # requests 0 and 2 share pages
    q = torch.randn(4, 8 * 64, generator=gen).to(torch.bfloat16).to(DEV)
    q[3] = q[0]
    out = torch.full_like(q, 7.0)
    step = step_of([1, 0, 1], [40, 3, 40])
    q2 = torch.cat([q[:1], q[:1]])
    kv8.paged_attention(q2, 8, 2, 64, pages, bt, 0.125, 0, out, step)
    assert torch.equal(out[0], out[1]) and bool((out[2:] == 7.0).all()) and not bool((out[0] == 7.0).all())
    step = step_of([0, 0, 0], [1, 2, 3])
    out.fill_(7.0)
    kv8.paged_attention(q, 8, 2, 64, pages, bt, 0.125, 0, out, step)
    assert bool((out == 7.0).all())


def test_a_page_id_outside_the_pool_sets_the_status_word_and_touches_nothing():
    from gibbs_b200.ops import kv8
    gen = torch.Generator().manual_seed(2)
    for dt in (torch.bfloat16, torch.float32):
        for portions, behind in (([1, 1], [20, 3]), ([40, 20], [0, 0])):
            pages = make_pages(4, 2, 16, 64, gen)
            before = [bits(t).clone() for t in pages.tensors()]
            bt = torch.full((2, 4), 1 << 20, dtype=torch.int32, device=DEV)
            bt[1] = -1
            n = sum(portions)
            x = torch.randn(n, 12 * 64, generator=gen).to(dt).to(DEV)
            q, step = torch.empty(n, 8 * 64, dtype=dt, device=DEV), step_of(portions, behind)
            kv8.qk_norm_rope_store(x, q, 8, 2, 64, None, None, EPS, None, 0, False, step, bt, pages)
            assert int(step.status.item()) == 1
            step.status.zero_()
            assert all(torch.equal(bits(a), b) for a, b in zip(pages.tensors(), before))
            kv8.paged_attention(q, 8, 2, 64, pages, bt, 0.125, 0, torch.empty_like(q), step)
            assert int(step.status.item()) == 2
            step.status.zero_()


@pytest.mark.parametrize("case", [ATTENTIONS[i] for i in (1, 2, 4, 6, 11, 21)])
def test_the_same_call_twice_and_in_a_graph_gives_the_same_bits(case):
    from gibbs_b200.ops import kv8
    dtype, heads, kv_heads, hd, page, window, portions, behind = case
    gen = torch.Generator().manual_seed(4)
    dt = torch.bfloat16 if dtype == "bf16" else torch.float32
    n_pages, bt = tables(portions, behind, page, random.Random(1))
    bt, n, step = bt.to(DEV), sum(portions), step_of(portions, behind)
    x = torch.randn(n, (heads + 2 * kv_heads) * hd, generator=gen).to(dt).to(DEV)

    def once(pages, q, out):
        kv8.qk_norm_rope_store(x, q, heads, kv_heads, hd, None, None, EPS, None, 0, False, step, bt, pages)
        kv8.paged_attention(q, heads, kv_heads, hd, pages, bt, hd ** -0.5, window, out, step)

    def fresh():
        return (make_pages(n_pages, kv_heads, page, hd, torch.Generator().manual_seed(8)),
                torch.zeros(n, heads * hd, dtype=dt, device=DEV), torch.zeros(n, heads * hd, dtype=dt, device=DEV))

    a, b, c = fresh(), fresh(), fresh()
    once(*a)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):                                   # another stream
        once(*b)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        once(*c)
    graph.replay()
    graph.replay()                                                    # (storing the same rows again changes nothing)
    torch.cuda.synchronize()
    for x1, y1, z1 in zip(a[0].tensors() + a[1:], b[0].tensors() + b[1:], c[0].tensors() + c[1:]):
        assert torch.equal(bits(x1), bits(y1)) and torch.equal(bits(x1), bits(z1))


def test_a_cache_larger_than_32_bit_offsets():
    """Pages behind the first 4 GB of a pool."""
    from gibbs_b200.ops import kv8
    n_pages, kv_heads, page, hd = 36000, 8, 128, 128                   # 4.7 GB each of keys and values
    k, v = (torch.zeros(n_pages, kv_heads, page, hd, dtype=torch.uint8, device=DEV).view(F8) for _ in range(2))
    pages = kv8.Pages(k, v, torch.ones(n_pages, kv_heads, device=DEV), torch.ones(n_pages, kv_heads, device=DEV))
    ids = [35999, 35000, 34000, 33001, 35998]
    for portions, behind in (([1], [600]), ([601], [0])):
        n = sum(portions)
        gen = torch.Generator().manual_seed(1)
        x = torch.randn(601, (16 + 16) * hd, generator=gen).to(torch.bfloat16)
        bt = torch.tensor([ids], dtype=torch.int32, device=DEV)
        q = torch.empty(601, 16 * hd, dtype=torch.bfloat16, device=DEV)
        kv8.qk_norm_rope_store(x.to(DEV), q, 16, 8, hd, None, None, EPS, None, 0, False, step_of([601], [0]), bt, pages)
        q = x[-n:, :16 * hd].contiguous().to(DEV)
        out = torch.empty_like(q)
        step = step_of(portions, behind)
        kv8.paged_attention(q, 16, 8, hd, pages, bt, hd ** -0.5, 0, out, step)
        assert int(step.status.item()) == 0
        keys, values = ((pages.k if i == 0 else pages.v)[ids].float() * (pages.k_scales if i == 0 else pages.v_scales)[ids][:, :, None, None]
                        for i in range(2))
        for h in range(8):
            kk, vv = (t[:, h].reshape(-1, hd)[:601].double().cpu() for t in (keys, values))
            want, weight, _ = plain.attention(q[-1:].double().cpu().view(1, 8, 2, hd)[:, h], kk, vv, hd ** -0.5, 0, [600])
            got = out[-1:].double().cpu().view(1, 8, 2, hd)[:, h]
            assert bool(((got - want).abs() <= 2.0 ** -7 * weight + 2.0 ** -14).all())


# ---------------------------------------------------------------------------------------------------
def test_refusals():
    from gibbs_b200.ops import KernelError, kv8
    pages = make_pages(4, 2, 16, 64, torch.Generator().manual_seed(0))
    step, bt = step_of([3], [0]), torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    x = torch.zeros(3, 8 * 64, dtype=torch.bfloat16, device=DEV)
    q = torch.zeros(3, 4 * 64, dtype=torch.bfloat16, device=DEV)
    store = lambda **k: kv8.qk_norm_rope_store(*[k.get(n, d) for n, d in (                             # noqa: E731
        ("x", x), ("q", q), ("heads", 4), ("kv", 2), ("hd", 64), ("qg", None), ("kg", None), ("eps", EPS), ("table", None), ("rd", 0),
        ("adj", False), ("step", step), ("bt", bt), ("pages", pages))])
    attend = lambda **k: kv8.paged_attention(*[k.get(n, d) for n, d in (                               # noqa: E731
        ("q", q), ("heads", 4), ("kv", 2), ("hd", 64), ("pages", pages), ("bt", bt), ("scale", 0.125), ("window", 0),
        ("out", torch.empty_like(q)), ("step", step))])
    store(), attend()
    for bad in (dict(x=x.half()), dict(x=x[:, :100]), dict(x=x[:2]), dict(q=q.float()), dict(q=q[:, :64]), dict(q=q[:2]), dict(hd=60),
                dict(hd=32), dict(heads=0), dict(qg=torch.ones(63, device=DEV)), dict(kg=torch.ones(64, device=DEV).double()),
                dict(table=torch.ones(33, device=DEV), rd=66), dict(bt=bt.long()), dict(bt=bt[:0]), dict(x=x.cpu()), dict(bt=bt.cpu()),
                dict(x=torch.zeros(8 * 64, 3, dtype=torch.bfloat16, device=DEV).T)):
        with pytest.raises(KernelError):
            store(**bad)
    for bad in (dict(q=q.half()), dict(heads=3), dict(kv=4), dict(hd=128), dict(q=q[:2]), dict(window=-1), dict(window=None), dict(bt=bt.long()),
                dict(bt=bt[0]), dict(out=torch.empty(3, 4 * 64, device=DEV)), dict(out=torch.empty(2, 4 * 64, dtype=torch.bfloat16, device=DEV)),
                dict(q=q.cpu())):
        with pytest.raises(KernelError):
            attend(**bad)


def test_tables_that_do_not_hold_the_contexts_and_rows_over_one_another_are_refused():
    from gibbs_b200.ops import KernelError, kv8
    pages = make_pages(4, 2, 16, 64, torch.Generator().manual_seed(0))
    q = torch.zeros(3, 4 * 64, dtype=torch.bfloat16, device=DEV)
    x = torch.zeros(3, 8 * 64, dtype=torch.bfloat16, device=DEV)
    bt = torch.zeros(1, 2, dtype=torch.int32, device=DEV)
    for portions, behind in (([3], [30]), ([1], [32])):
        with pytest.raises(KernelError, match="do not hold"):
            kv8.qk_norm_rope_store(x, q, 4, 2, 64, None, None, EPS, None, 0, False, step_of(portions, behind), bt, pages)
        with pytest.raises(KernelError, match="do not hold"):
            kv8.paged_attention(q, 4, 2, 64, pages, bt, 0.125, 0, torch.empty_like(q), step_of(portions, behind))
    with pytest.raises(KernelError, match="over one another"):
        kv8.paged_attention(q, 4, 2, 64, pages, bt, 0.125, 0, q[:1].clone().expand(3, -1), step_of([3], [29]))
    kv8.paged_attention(q[:1].expand(3, -1), 4, 2, 64, pages, bt, 0.125, 0, torch.empty_like(q), step_of([3], [29]))
    # (rows of q alone need no pages, so no table that holds them)
    kv8.qk_norm_rope_store(x, q, 4, 2, 64, None, None, EPS, None, 0, False, step_of([3], [300]), bt, None)


WAYS = [(torch.bfloat16, [1, 1], 64, 16), (torch.bfloat16, [40, 2], 64, 16), (torch.bfloat16, [40], 128, 64), (torch.float32, [1, 3], 64, 16),
        (torch.float32, [5], 48, 5)]


@pytest.mark.parametrize("dt,portions,hd,page", WAYS)
def test_windows_that_no_context_reaches(dt, portions, hd, page):
    from gibbs_b200.ops import kv8
    gen = torch.Generator().manual_seed(3)
    behind = [100] * len(portions)
    n_pages, bt = tables(portions, behind, page, random.Random(1))
    pages = make_pages(n_pages, 2, page, hd, gen)
    q = torch.randn(sum(portions), 4 * hd, generator=gen).to(dt).to(DEV)
    outs = [kv8.paged_attention(q, 4, 2, hd, pages, bt.to(DEV), hd ** -0.5, w, torch.empty_like(q), step_of(portions, behind))
            for w in (0, 2 ** 31 - 1, 2 ** 31 - 100, 2 ** 30, 2 ** 32 + 5, 2 ** 62)]
    for o in outs[1:]:
        assert torch.equal(o, outs[0])


@pytest.mark.parametrize("dt,portions,hd,page", WAYS)
@pytest.mark.parametrize("bad", [-2 ** 31, -2 ** 31 + 2, -7, 2 ** 31 - 1])
def test_page_ids_far_outside(dt, portions, hd, page, bad):
    from gibbs_b200.ops import kv8
    gen = torch.Generator().manual_seed(3)
    behind = [100] * len(portions)
    n_pages, bt = tables(portions, behind, page, random.Random(1))
    pages = make_pages(n_pages, 2, page, hd, gen)
    q = torch.randn(sum(portions), 4 * hd, generator=gen).to(dt).to(DEV)
    bt[0, 2] = bad
    step = step_of(portions, behind)
    kv8.paged_attention(q, 4, 2, hd, pages, bt.to(DEV), hd ** -0.5, 0, torch.empty_like(q), step)
    assert int(step.status.item()) == 2
    step.status.zero_()
    before = [bits(t).clone() for t in pages.tensors()]
    bt[:, 100 // page:] = bad
    x = torch.randn(sum(portions), 8 * hd, generator=gen).to(dt).to(DEV)
    kv8.qk_norm_rope_store(x, q, 4, 2, hd, None, None, EPS, None, 0, False, step, bt.to(DEV), pages)
    assert int(step.status.item()) == 1
    step.status.zero_()
    assert all(torch.equal(bits(a), b) for a, b in zip(pages.tensors(), before))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_more_requests_than_a_grid_has_rows(dt):
    """70,001 requests of one token each: a token that sees itself alone gets its own value."""
    from gibbs_b200.ops import kv8
    n, hd = 70001, 64
    gen = torch.Generator().manual_seed(9)
    x = torch.randn(n, 4 * hd, generator=gen).to(dt).to(DEV)
    pages = make_pages(n, 1, 16, hd, gen)
    bt = torch.randperm(n, generator=gen).to(torch.int32).view(n, 1).to(DEV)
    q, step = torch.empty(n, 2 * hd, dtype=dt, device=DEV), step_of([1] * n, [0] * n)
    kv8.qk_norm_rope_store(x, q, 2, 1, hd, None, None, EPS, None, 0, False, step, bt, pages)
    assert torch.equal(q, x[:, :2 * hd])
    out = kv8.paged_attention(q, 2, 1, hd, pages, bt, 0.125, 0, torch.empty_like(q), step)
    held = pages.dequantized()[1][bt[:, 0].long(), 0, 0]
    half, smallest = 2.0 ** -4, 2.0 ** -10 * pages.v_scales[bt[:, 0].long()]
    assert bool(((held - x[:, 3 * hd:].float()).abs() <= torch.maximum(half * x[:, 3 * hd:].float().abs(), smallest)).all())
    # one weight over itself: 2^-11 for it in 16 bits, 2^-22 for it and for the quotient, and the output's own rounding
    tol = (2.0 ** -11 + 2.0 ** -9 if dt == torch.bfloat16 else 0.0) + 2.0 ** -20
    assert bool(((out.float().view(n, 2, hd) - held[:, None]).abs() <= tol * held[:, None].abs()).all())


def test_calls_on_two_streams_at_once():
    from gibbs_b200.ops import kv8
    gen = torch.Generator().manual_seed(4)
    calls = []
    for portions, behind, hd, page in (([1] * 4, [9000, 8000, 100, 5], 128, 64), ([300, 1, 1], [4000, 3000, 17], 64, 16)):
        n_pages, bt = tables(portions, behind, page, random.Random(1))
        q = torch.randn(sum(portions), 8 * hd, generator=gen).to(torch.bfloat16).to(DEV)
        calls.append((q, 8, 2, hd, make_pages(n_pages, 2, page, hd, gen), bt.to(DEV), hd ** -0.5, 0, torch.empty_like(q), step_of(portions, behind)))
    want = [kv8.paged_attention(*c).clone() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, c in zip(streams, calls):
            with torch.cuda.stream(s):
                kv8.paged_attention(*c)
    torch.cuda.synchronize()
    for c, w in zip(calls, want):
        assert torch.equal(c[8], w) and int(c[9].status.item()) == 0


# ---------------------------------------------------------------------------------------------------
def copy_groups(rows, gen):
    whole = torch.randint(0, 256, (rows + 2, 4096 * 5 + 64), dtype=torch.uint8, generator=gen).to(DEV)
    strided = whole[1:-1, :4096 * 5 + 48]
    odd = torch.randint(0, 256, (rows, 37), dtype=torch.uint8, generator=gen).to(DEV)
    words = torch.randn(rows, 3, generator=gen).to(DEV)
    pages = torch.randn(rows, 4, 16, 64, generator=gen).to(F8).to(DEV)
    return [strided, odd, words, pages], whole


@pytest.mark.parametrize("n", [0, 1, 7, 440, 441, 1500])
def test_row_copies(n):
    from gibbs_b200.ops import RowCopies
    gen = torch.Generator().manual_seed(n)
    rows = 2 * n + 3
    first, whole = copy_groups(rows, gen)
    second = [torch.randn(5, 1000, generator=gen).bfloat16().to(DEV)]
    ids = torch.randperm(rows, generator=gen)[:2 * n].tolist()
    pairs = list(zip(ids[:n], ids[n:]))
    if n > 1:
        pairs[1] = (pairs[0][0], pairs[1][1])                    # one source for two
    copies = RowCopies([first, second])
    for given in (pairs, torch.tensor(pairs, dtype=torch.int32).reshape(-1, 2)):
        want = [bits(t).clone() for t in first + second]
        whole_before = whole.clone()
        for s, d in pairs:
            for w in want[:4]:
                w[d] = w[s]
        want[4][4] = want[4][0]
        copies.copy([given, [(0, 4)]])
        for t, w in zip(first + second, want):
            assert torch.equal(bits(t), w)
        whole_before[1:-1, :4096 * 5 + 48] = want[0]
        assert torch.equal(whole, whole_before)                  # nothing outside the rows
    assert copies.copy([[], []]) == 0


def test_row_copies_refusals_leave_everything_as_it_was():
    from gibbs_b200.ops import KernelError, RowCopies
    t = torch.arange(40, device=DEV).float().view(10, 4)
    before = t.clone()
    copies = RowCopies([[t]])
    for pairs in ([[(0, 10)]], [[(-1, 2)]], [[(3, 3)]], [[(0, 1), (2, 1)]], [[(0, 1), (1, 2)]], [[(1, 2), (0, 1)]], [[(0, 1)], []], [[(1 << 40, 0)]],
                  [torch.tensor([[0, 1]], device=DEV, dtype=torch.int32)], [torch.tensor([[0, 1]])], [torch.tensor([0, 1], dtype=torch.int32)]):
        with pytest.raises(KernelError):
            copies.copy(pairs)
    assert torch.equal(t, before)
    for groups in ([], [[]], [[t.cpu()]], [[t, torch.zeros(9, 4, device=DEV)]], [[t.T.contiguous().T]], [[t]] * 17,
                   [[torch.zeros(4, device=DEV).expand(10, 4)]]):
        with pytest.raises(KernelError):
            RowCopies(groups)


def test_row_copies_on_another_stream_and_in_a_graph():
    from gibbs_b200.ops import RowCopies
    t = torch.arange(4000, device=DEV).float().view(10, 400)
    copies = RowCopies([[t]])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copies.copy([[(0, 1), (0, 2)]])
    t[0] = -1.0
    graph.replay()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        copies.copy([[(1, 9)]])
    torch.cuda.synchronize()
    assert bool((t[[1, 2, 9]] == -1).all()) and float(t[3, 0]) == 1200
