"""A paged cache held in 8 bits and what works on it: storing a step's keys and values, attention of single tokens and of
prompt portions over it, and copying its pages when a request is forked.

The cache.  Keys and values lie in pages ``[n_pages, kv_heads, page_size, head_dim]`` of e4m3 numbers with one scale for
each page and kv head, a power of two: an entry stands for number * scale.  A scale is the smallest 2^e, e >= -64, that
holds the page's largest magnitude within 448; it only grows while a page fills, and when it grows the rows that the page
held already are rounded again under the new one.

``store``      q, k, v rows [tokens, (heads + 2 kv_heads) * head_dim]: a norm per head (RMS, with a gain) and a rotation by
               the position of q and k, then k and v into the pages.  Out: the rotated q, the pages and their scales.
``attention``  out = softmax(scale * q K^T over the visible keys) V, query head h on kv head h // (heads / kv_heads); a key j
               is visible to position p when p - window < j <= p (window 0: j <= p).
``copy``       rows ``src`` of every tensor of a cache into rows ``dst``.

Sizes are those of this repository's configurations and benchmark, or generic.
"""
from __future__ import annotations

import math

import torch

own = False

F64 = torch.float64
E4M3 = torch.float8_e4m3fn
EPS = 1e-5
THETA = 1000000.0
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
LARGEST_SCORES = 16 * 8192 * 8192           # (query head, key) pairs of the largest prompt, what a drawn one stays below
LARGEST_KEYS = 4 * 32768 * 8 * 128          # values of the largest cache of keys


def listed():
    return [
        # a decode step of a server's small batch, just after prompts of 2,048 tokens: every request stores one token
        dict(name="store_decode_batch8", op="store", type="bf16", heads=32, kv_heads=8, dim=64, page=16, portions="8*1",
             behind="2048,2050,2063,2055,2049,2061,2058,2052"),
        # a whole prompt in one step
        dict(name="store_prompt_2048", op="store", type="bf16", heads=32, kv_heads=8, dim=64, page=16, portions="2048",
             behind="0"),
        # the 32-bit path: prompt portions and single tokens in one step, pages that begin and end inside a portion
        dict(name="store_ragged_f32", op="store", type="f32", heads=16, kv_heads=2, dim=128, page=64,
             portions="700,1,333,65,1", behind="0,1500,77,4000,63"),
        # one user, one token after a prompt of 2,048
        dict(name="decode_one_2048", op="attention", type="bf16", heads=32, kv_heads=8, dim=64, page=16, portions="1",
             behind="2047", window=0),
        # a full batch of a server
        dict(name="decode_batch64_2048", op="attention", type="bf16", heads=32, kv_heads=8, dim=64, page=16,
             portions="64*1", behind="64*2111", window=0),
        # few users with long documents
        dict(name="decode_four_long", op="attention", type="bf16", heads=32, kv_heads=8, dim=128, page=64, portions="4*1",
             behind="32767,32100,31007,29999", window=0),
        # the 32-bit path, requests of every length, heads in groups of three
        dict(name="decode_ragged_f32", op="attention", type="f32", heads=24, kv_heads=8, dim=64, page=16, portions="9*1",
             behind="0,1,15,16,130,999,2500,4001,511", window=0),
        # a whole prompt in one step
        dict(name="prompt_2048", op="attention", type="bf16", heads=32, kv_heads=8, dim=64, page=16, portions="2048",
             behind="0", window=0),
        # a long prompt with wide heads
        dict(name="prompt_8192_wide", op="attention", type="bf16", heads=16, kv_heads=4, dim=128, page=64, portions="8192",
             behind="0", window=0),
        # a server's step: a portion of a long prompt, a short prompt, and single tokens beside them, with a window
        dict(name="portions_and_tokens", op="attention", type="bf16", heads=24, kv_heads=8, dim=64, page=16,
             portions="500,1,1,1,37", behind="7500,2060,511,15,0", window=4096),
        # a second answer to a prompt: the page that both will write on, and the state of the layers without pages
        dict(name="fork_one", op="copy", layers=6, kv_heads=8, dim=64, page=16, pairs=1, state=163840),
        # many requests move at once (a search over beams): a thousand pages of six layers
        dict(name="copy_1000_pages", op="copy", layers=6, kv_heads=8, dim=64, page=16, pairs=1000, state=0),
    ]


# ---------------------------------------------------------------------------------------------------
# sizes of a case
# ---------------------------------------------------------------------------------------------------

def _numbers(text):
    out = []
    for part in str(text).split(","):
        n, _, v = part.rpartition("*")
        out += [int(v)] * (int(n) if n else 1)
    return out


def _text(numbers):
    return ",".join(str(n) for n in numbers)


def _spread(rng, lo, hi):
    """A whole number in lo..hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def _layout(rng):
    heads, kv_heads = rng.choice([(32, 8), (24, 8), (16, 4), (16, 2), (12, 12), (8, 1), (40, 8), (14, 2)])
    return dict(heads=heads, kv_heads=kv_heads, dim=rng.choice([64, 64, 128]), page=rng.choice([16, 16, 32, 64, 128]))


def draw(rng):
    op = rng.choice(["store", "store", "attention", "attention", "attention", "attention", "copy"])
    if op == "copy":
        return dict(op="copy", layers=rng.randint(1, 12), kv_heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 128]),
                    page=rng.choice([16, 32, 64]), pairs=_spread(rng, 1, 250), state=rng.choice([0, 4096, 24592, 163840]))
    kind = "f32" if rng.random() < 0.2 else "bf16"
    size = _layout(rng)
    if op == "store":
        if rng.random() < 0.4:
            n = _spread(rng, 1, 64)
            portions, behind = [1] * n, [_spread(rng, 1, 8192) - 1 for _ in range(n)]
        else:
            portions = [_spread(rng, 1, 2048) for _ in range(rng.randint(1, 4))]
            behind = [rng.choice([0, _spread(rng, 1, 8192)]) for _ in portions]
        return dict(op="store", type=kind, portions=_text(portions), behind=_text(behind), **size)
    window = rng.choice([0, 0, 0, _spread(rng, 64, 8192)])
    if rng.random() < 0.5:
        n = _spread(rng, 1, 64)
        most = min(32768, LARGEST_KEYS // (n * size["kv_heads"] * size["dim"]))
        behind = [_spread(rng, 1, most) - 1 for _ in range(n)]
        return dict(op="attention", type=kind, portions=_text([1] * n), behind=_text(behind), window=window, **size)
    portions = [_spread(rng, 1, 4096) for _ in range(rng.randint(1, 3))]
    behind = [rng.choice([0, _spread(rng, 1, 8192)]) for _ in portions]
    while len(portions) * max(portions) * size["heads"] * max(p + b for p, b in zip(portions, behind)) > LARGEST_SCORES // 2:
        portions = [max(1, p // 2) for p in portions]
        behind = [b // 2 for b in behind]
    return dict(op="attention", type=kind, portions=_text(portions), behind=_text(behind), window=window, **size)


def _first_key(position, window):
    return max(0, position - window + 1) if window else 0


def work(case):
    if case["op"] == "copy":
        page = case["kv_heads"] * case["page"] * case["dim"] + 4 * case["kv_heads"]
        return {"bytes": 2 * (case["pairs"] * 2 * case["layers"] * page + case["state"]), "flops": 0}
    portions, behind = _numbers(case["portions"]), _numbers(case["behind"])
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    size, n = (2 if case["type"] == "bf16" else 4), sum(portions)
    if case["op"] == "store":
        # the rows in, q out, k and v out in 8 bits; a norm, a rotation and a scaling of every value
        return {"bytes": n * (heads + 2 * kv_heads) * dim * size + n * heads * dim * size + n * 2 * kv_heads * dim,
                "flops": 10 * n * (heads + 2 * kv_heads) * dim}
    keys = pairs = 0
    for p, b in zip(portions, behind):
        keys += b + p - _first_key(b, case["window"])
        if case["window"]:
            pairs += sum(min(case["window"], j + 1) for j in range(b, b + p))
        else:
            pairs += p * b + p * (p + 1) // 2
    return {"bytes": 2 * n * heads * dim * size + keys * 2 * kv_heads * dim, "flops": 4 * heads * dim * pairs}


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------

def _scale_of(largest):
    """The smallest power of two, 2^-64 at least, under which `largest` is 448 or less."""
    m, e = torch.frexp(largest.float())               # largest = m 2^e with m in [1/2, 1); 448 = 7/8 of 2^9
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-64)
    return torch.ldexp(torch.ones_like(largest, dtype=torch.float32), e)


def _bytes(t):
    return t.view(torch.uint8) if t.dtype == E4M3 else t


def _requests(case, gen, dev):
    """The step's requests as a server has them: where each begins, how long it is, and its pages."""
    portions, behind, page = _numbers(case["portions"]), _numbers(case["behind"]), case["page"]
    ends = [b + p for b, p in zip(behind, portions)]
    blocks = -(-max(ends) // page)
    table = torch.full((len(ends), blocks), -1, dtype=torch.int64)
    n_pages = sum(-(-e // page) for e in ends) + 3
    ids = torch.randperm(n_pages, generator=gen)
    at = 0
    for r, (b, e) in enumerate(zip(behind, ends)):
        first = _first_key(b, case.get("window", 0)) // page      # pages that the window has passed were given back
        have = -(-e // page)
        table[r, first:have] = ids[at + first:at + have]
        at += have
    starts = [sum(portions[:r]) for r in range(len(portions))]
    req = torch.cat([torch.full((p,), r, dtype=torch.int64) for r, p in enumerate(portions)])
    pos = torch.cat([torch.arange(b, b + p) for b, p in zip(behind, portions)])
    s = dict(portions=portions, behind=behind, ends=ends, n_pages=n_pages, table=table.to(dev), req=req.to(dev),
             pos=pos.to(dev), starts=torch.tensor(starts, device=dev))
    s["int"] = {k: v.to(torch.int32).to(dev) for k, v in dict(
        table=table, req=req, pos=pos, start=torch.tensor(starts), count=torch.tensor(portions),
        before=torch.tensor(behind), after=torch.tensor(ends)).items()}
    return s


def _step(s):
    """What the engine hands its layers in a step."""
    from gibbs_b200 import ops
    from gibbs_b200.engine.step import StepState
    i = s["int"]
    return StepState(n_tokens=int(i["req"].numel()), n_requests=len(s["portions"]), n_want=0, token_ids=i["req"],
                     tok_req=i["req"], tok_pos=i["pos"], q_start=i["start"], q_len=i["count"], start_pos=i["before"],
                     ctx_len=i["after"], want_rows=i["start"][:0], status=ops.device_status(i["req"].device),
                     max_q_len=max(s["portions"]), max_ctx_len=max(s["ends"]))


def prepare(case, seed):
    dev = torch.device("cuda")
    host = torch.Generator().manual_seed(seed)
    gen = torch.Generator(device=dev).manual_seed(seed)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=dev)                              # noqa: E731
    kv_heads, dim, page = case["kv_heads"], case["dim"], case["page"]
    if case["op"] == "copy":
        n_pages = 2 * case["pairs"] + 7
        ids = torch.randperm(n_pages, generator=host)[:2 * case["pairs"]]
        src, dst = ids[:case["pairs"]], ids[case["pairs"]:]
        pages = []
        for _ in range(2 * case["layers"]):
            pages += [randn(n_pages, kv_heads, page, dim).to(E4M3),
                      torch.ldexp(torch.ones(n_pages, kv_heads, device=dev),
                                  torch.randint(-12, 4, (n_pages, kv_heads), generator=gen, device=dev))]
        slots = []
        if case["state"]:
            slots = [torch.randint(0, 256, (4, case["state"]), generator=gen, device=dev, dtype=torch.uint8)]
        s = dict(case=case, pages=pages, slots=slots, src=src.to(dev), dst=dst.to(dev),
                 pairs=torch.stack([src, dst], 1).to(torch.int32))
        if own:
            from gibbs_b200.ops import RowCopies
            s["copies"] = RowCopies([pages, slots] if slots else [pages])
        return s
    dtype, heads = TYPES[case["type"]], case["heads"]
    s = dict(_requests(case, host, dev), case=case)
    n_pages, n = s["n_pages"], int(s["req"].numel())
    # keys behind a norm and a rotation have about one size; values differ from head to head
    for name in ("k", "v"):
        values = randn(n_pages, kv_heads, page, dim)
        if name == "v":
            values *= torch.exp(0.5 * randn(1, kv_heads, 1, 1))
        if case["op"] == "store":
            values *= 0.7                                      # (some scales grow when the page's next rows come)
        scale = _scale_of(values.abs().amax(dim=(2, 3)))
        s[name + "_scale"] = scale
        s[name] = (values / scale[:, :, None, None]).to(E4M3)
        del values
    if case["op"] == "store":
        s["qkv"] = randn(n, (heads + 2 * kv_heads) * dim).to(dtype)
        s["q_out"] = torch.empty(n, heads * dim, dtype=dtype, device=dev)
        s["q_gain"], s["k_gain"] = (1 + 0.1 * randn(dim) for _ in range(2))
        freq = THETA ** (-torch.arange(0, dim, 2, device=dev, dtype=F64) / dim)
        s["rotary"] = torch.cat([freq, torch.ones(1, device=dev, dtype=F64)]).float()    # (the last: a factor on cos and sin)
        # the pages that get rows, how many rows each held before, and each token's page among them
        page_of = s["table"][s["req"], s["pos"] // page]
        s["touched"], s["which"] = torch.unique(page_of, return_inverse=True)
        held = torch.full((len(s["touched"]),), page, device=dev, dtype=torch.int64)
        s["held"] = held.scatter_reduce(0, s["which"], s["pos"] % page, "amin")
        got = torch.zeros_like(held).scatter_add(0, s["which"], torch.ones_like(s["which"]))
        s["filled"] = s["held"] + got
    else:
        # queries behind the same norm and rotation; a few heads look sharply at a few keys
        s["q"] = (randn(n, heads * dim) * torch.exp(0.3 * randn(1, heads, 1)).expand(1, heads, dim).reshape(1, -1)).to(dtype)
        s["out"] = torch.empty(n, heads * dim, dtype=dtype, device=dev)
        s["scale"] = dim ** -0.5
    if own:
        from gibbs_b200.ops import kv8
        s["cache"] = kv8.Pages(s["k"], s["v"], s["k_scale"], s["v_scale"])
        s["step"] = _step(s)
    return s


# ---------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------

def run(state):
    return {"store": _store, "attention": _attention, "copy": _copy}[state["case"]["op"]](state)


def _copy(s):
    if own:
        s["copies"].copy([s["pairs"], [(1, 2)]] if s["slots"] else [s["pairs"]])
    else:
        for t in s["pages"]:
            _bytes(t)[s["dst"]] = _bytes(t)[s["src"]]
        for t in s["slots"]:
            t[2] = t[1]
    return {"pages": s["pages"], "slots": s["slots"]}


def _store(s):
    c = s["case"]
    heads, kv_heads, dim = c["heads"], c["kv_heads"], c["dim"]
    answer = {"k": s["k"], "v": s["v"], "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if own:
        from gibbs_b200.ops import kv8
        kv8.qk_norm_rope_store(s["qkv"], s["q_out"], heads, kv_heads, dim, s["q_gain"], s["k_gain"], EPS, s["rotary"], dim,
                               False, s["step"], s["int"]["table"], s["cache"])
        return dict(answer, q=s["q_out"])
    x = s["qkv"].float().view(-1, heads + 2 * kv_heads, dim)
    q, k, v = x.split([heads, kv_heads, kv_heads], dim=1)
    angle = s["pos"].to(F64)[:, None] * s["rotary"][:-1].to(F64)
    cos, sin = ((f(angle) * s["rotary"][-1]).float()[:, None, :] for f in (torch.cos, torch.sin))

    def normed_rotated(y, gain):
        y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * gain
        a, b = y[..., :dim // 2], y[..., dim // 2:]
        return torch.cat([a * cos - b * sin, a * sin + b * cos], -1)

    for name, rows in (("k", normed_rotated(k, s["k_gain"])), ("v", v)):
        _append(_bytes(s[name]), s[name + "_scale"], rows, s)
    return dict(answer, q=normed_rotated(q, s["q_gain"]).reshape(-1, heads * dim).to(s["qkv"].dtype))


def _append(pages, scales, rows, s):
    """Rows [tokens, kv_heads, dim] into the pages they belong to, in place."""
    page, touched = s["case"]["page"], s["touched"]
    now = pages[touched]                                                        # [touched, kv_heads, page, dim], as bytes
    new = torch.zeros(now.shape, device=rows.device)
    new[s["which"], :, s["pos"] % page] = rows
    at = torch.arange(page, device=rows.device)[None, :]
    is_old, is_new = at < s["held"][:, None], (at >= s["held"][:, None]) & (at < s["filled"][:, None])
    before = torch.where(s["held"][:, None] > 0, scales[touched], torch.zeros_like(scales[touched]))
    after = torch.maximum(before, _scale_of(new.abs().amax(dim=(2, 3))))
    old = now.view(E4M3).float() * (before / after)[:, :, None, None]
    values = torch.where(is_new[:, None, :, None], new / after[:, :, None, None], old).to(E4M3).view(torch.uint8)
    pages[touched] = torch.where((is_old | is_new)[:, None, :, None], values, now)
    scales[touched] = after


def _attention(s):
    c = s["case"]
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    if own:
        from gibbs_b200.ops import kv8
        return kv8.paged_attention(s["q"], heads, kv_heads, dim, s["cache"], s["int"]["table"], s["scale"], c["window"],
                                   s["out"], s["step"])
    group, n_req, most = heads // kv_heads, len(s["portions"]), max(s["portions"])
    table = s["table"].clamp(min=0)
    keys, values = (
        (_bytes(s[name])[table].view(E4M3).float() * s[name + "_scale"][table][..., None, None])
        .permute(0, 2, 1, 3, 4).reshape(n_req, kv_heads, -1, dim) for name in ("k", "v"))
    # queries of all requests side by side: [requests, kv_heads, group * portion, dim]
    within = torch.arange(most, device=table.device)
    count = s["int"]["count"][:, None]
    rows = (s["starts"][:, None] + within).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float().view(-1, kv_heads, group, dim)[rows].permute(0, 2, 3, 1, 4).reshape(n_req, kv_heads, group * most, dim)
    scores = (q @ keys.transpose(2, 3)).mul_(s["scale"]).view(n_req, kv_heads, group, most, -1)
    pos = (s["int"]["before"][:, None] + within)[:, :, None]
    at = torch.arange(keys.shape[2], device=table.device)
    seen = at <= pos
    if c["window"]:
        seen = seen & (at > pos - c["window"])
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    weights = scores.exp_()
    total = weights.sum(-1, keepdim=True)
    out = (weights.view(n_req, kv_heads, group * most, -1) @ values).view(n_req, kv_heads, group, most, dim)
    out = (out / total).permute(0, 3, 1, 2, 4).reshape(n_req, most, heads * dim)
    return out[within < count].to(s["q"].dtype)


# ---------------------------------------------------------------------------------------------------
# in 64 bits, from the definitions
# ---------------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"store": _exact_store, "attention": _exact_attention, "copy": _exact_copy}[case["op"]](s)


def _exact_copy(s):
    """(Moved, not computed.)"""
    for t in s["pages"] + s["slots"]:
        b = _bytes(t)
        for x, y in (s["pairs"].tolist() if t.dim() != 2 or t.dtype != torch.uint8 else [(1, 2)]):
            b[y].copy_(b[x])
    return {"pages": s["pages"], "slots": s["slots"]}


def _exact_store(s):
    """The pages' numbers before they are rounded to 8 bits, request by request and page by page."""
    c = s["case"]
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    x = s["qkv"].to(F64).reshape(-1, heads + 2 * kv_heads, dim)
    freq, factor = s["rotary"][:-1].to(F64), float(s["rotary"][-1])
    turn = torch.exp(1j * s["pos"].to(F64)[:, None] * freq)[:, None, :] * factor
    done = []
    for part, gain in ((x[:, :heads], s["q_gain"]), (x[:, heads:heads + kv_heads], s["k_gain"])):
        y = part / torch.sqrt(part.pow(2).sum(-1, keepdim=True) / dim + EPS) * gain.to(F64)
        z = torch.complex(y[..., :dim // 2].contiguous(), y[..., dim // 2:].contiguous()) * turn
        done.append(torch.cat([z.real, z.imag], -1))
    answer = {"q": done[0].reshape(-1, heads * dim)}
    for name, rows in (("k", done[1]), ("v", x[:, heads + kv_heads:])):
        numbers, scales = s[name].to(F64), s[name + "_scale"].to(F64)
        row = 0
        for r, (b, p) in enumerate(zip(s["behind"], s["portions"])):
            at = b
            while at < b + p:
                n = min(page - at % page, b + p - at)
                i, o = int(s["table"][r, at // page]), at % page
                new = rows[row:row + n].transpose(0, 1)                                # [kv_heads, n, dim]
                need = torch.exp2(torch.ceil(torch.log2(new.abs().amax(dim=(1, 2)) / 448)).clamp(min=-64))
                if o:
                    need = torch.maximum(need, scales[i])
                    numbers[i, :, :o] *= (scales[i] / need)[:, None, None]
                numbers[i, :, o:o + n] = new / need[:, None, None]
                scales[i] = need
                at, row = at + n, row + n
        answer[name], answer[name + "_scale"] = numbers, scales
    return answer


def _exact_attention(s):
    c = s["case"]
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    group = heads // kv_heads
    out = torch.empty(s["q"].shape, dtype=F64, device=s["q"].device)
    row = 0
    for r, (b, p) in enumerate(zip(s["behind"], s["portions"])):
        low = _first_key(b, c["window"])
        ids = s["table"][r, low // page:-(-(b + p) // page)]
        for h in range(kv_heads):
            k, v = ((s[n].view(torch.uint8)[ids, h].view(E4M3).to(F64) * s[n + "_scale"][ids, h].to(F64)[:, None, None])
                    .reshape(-1, dim) for n in ("k", "v"))
            key = low // page * page + torch.arange(k.shape[0], device=k.device)
            for g in range(h * group, (h + 1) * group):
                for i in range(0, p, 2048):
                    n = min(2048, p - i)
                    at = torch.arange(b + i, b + i + n, device=k.device)[:, None]
                    logits = s["q"][row + i:row + i + n, g * dim:(g + 1) * dim].to(F64) @ k.T * s["scale"]
                    hidden = (key > at) | ((key <= at - c["window"]) if c["window"] else (key < 0))
                    w = torch.softmax(logits.masked_fill(hidden, -math.inf), -1)
                    out[row + i:row + i + n, g * dim:(g + 1) * dim] = w @ v
        row += p
    return out
