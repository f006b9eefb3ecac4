"""The engine with keys and values held in 8 bits, and forked requests, against the plain implementation: whole prompts, portions,
single tokens, mixed steps; layers with a window and layers that read another's cache; step plans, graphs and plain forwards."""
import math

import numpy as np
import pytest
import torch

import plain_kv8
import plain_lfm2 as plain
from helpers import (TINY, first_wrong, make_folder, plain_logits, random_ids, rel_err, run_trace_on_engine, sharpen_attention,
                     trace_mixed, trace_portions, trace_tail_decoded, trace_whole)

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
DTYPES = ["float32", "bfloat16"]
PAGE = 16

# Against an oracle that holds its keys and values in the same 8 bits, what is left are numbers that fall to the other side of a tie:
# in float32 those within 2^-20 of one, 2^-17 of all (a step is 2^-3), of some 10^5 numbers a few, and one of them turns a score by
# up to 2^-3 of one of its products: 5e-3 of a logits row.  In bfloat16 keys and values are 2^-8 off before they are rounded, so one
# in 2^5 takes the next number, a whole step of 2^-3 away: sqrt(2^-5) 2^-3 = 2.2 % of a key or a value, root mean square.  (A first
# bound of 6 % took a step's rounding error, 2^-3 / sqrt(12), for the step itself.)  The four layers of the deepest model here add
# eight of these, its keys' and its values', in quadrature: sqrt(8) 2.2 % = 6.2 %, beside the 2 % that the plain cache is allowed:
# 8.2 %, and 10 % for the spread of the largest of a row's errors over the largest of its logits (two maxima of some 300 numbers,
# each 3 sigma give or take a tenth).
TOL8 = {"float32": 5e-3, "bfloat16": 1e-1}
_models = {}


def held_in_8_bits(x: torch.Tensor) -> torch.Tensor:
    """Rows [n, kv_heads, hd] as 8-bit pages of PAGE rows stand for them."""
    n, kvh, hd = x.shape
    blocks = -(-n // PAGE)
    pages = plain_kv8.PlainPages(torch.zeros(blocks, kvh, PAGE, hd), torch.zeros(blocks, kvh))
    for b in range(blocks):
        pages.store(b, 0, x[b * PAGE:(b + 1) * PAGE].cpu())
    held = pages.n * pages.s.abs()[:, :, None, None]
    return held.permute(0, 2, 1, 3).reshape(-1, kvh, hd)[:n].to(x)


@pytest.fixture
def oracle_in_8_bits(monkeypatch):
    whole = plain.causal_attention
    monkeypatch.setattr(plain, "causal_attention",
                        lambda q, k, v, *a, **b: whole(q, held_in_8_bits(k), held_in_8_bits(v), *a, **b))


def _model(tmp_path_factory, name, dtype):
    key = (name, dtype)
    if key not in _models:
        from gibbs_b200 import load_model
        stored = torch.bfloat16 if dtype == "bfloat16" else torch.float32
        folder = make_folder(tmp_path_factory.mktemp("kv8"), name, stored=stored)
        if name == "C":
            folder = sharpen_attention(folder)
        _models[key] = (folder, load_model(folder, dtype=dtype, device=DEV))
    return _models[key]


def _engine(model, **k):
    from gibbs_b200 import Engine
    return Engine(model, **{**dict(n_pages=64, page_size=PAGE, max_requests=4, max_step_tokens=512, guard_cache=True,
                                   cache_dtype="float8_e4m3"), **k})


def _requests(name, lengths, seed=0):
    return {f"r{i}": random_ids(seed * 100 + i, n, TINY[name][0]["vocab_size"]) for i, n in enumerate(lengths)}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name", ["A", "B", "C"])
def test_logits_under_every_way_of_cutting_the_work(tmp_path_factory, oracle_in_8_bits, name, dtype):
    folder, model = _model(tmp_path_factory, name, dtype)
    eng = _engine(model)
    assert eng.plan is not None and eng.use_graphs and eng.cache.in_8_bits
    reqs = _requests(name, [1, 7, 40, 150, 300])
    want = {rid: plain_logits(folder, ids) for rid, ids in reqs.items()}
    worst = 0.0
    for steps in (trace_whole(reqs), trace_tail_decoded(reqs), trace_portions(reqs), trace_mixed(reqs, capacity_tokens=640, seed=3)):
        got = run_trace_on_engine(eng, steps)
        for rid in reqs:
            bad = first_wrong(got[rid], want[rid], TOL8[dtype])
            assert bad is None, (rid, bad)
            worst = max(worst, rel_err(got[rid], want[rid]))
    assert eng.cache.free_pages() == [64]
    print(f"{name} {dtype}: worst rel err {worst:.3g}")


@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("C", "bfloat16"), ("C", "float32"), ("B", "bfloat16")])
def test_plans_graphs_and_plain_forwards_give_the_same_bits(tmp_path_factory, name, dtype):
    _, model = _model(tmp_path_factory, name, dtype)
    reqs = _requests(name, [33, 5, 64, 90], seed=2)
    steps = trace_mixed(reqs, capacity_tokens=640, seed=5) + trace_tail_decoded({"z" + k: v for k, v in reqs.items()}, tail=6)
    a = run_trace_on_engine(_engine(model), steps)
    b = run_trace_on_engine(_engine(model, use_graphs=False), steps)
    c = run_trace_on_engine(_engine(model, use_graphs=False, use_plan=False), steps)
    for rid in a:
        assert np.array_equal(b[rid], c[rid])
        # (a graph's launches are sized for the longest context, so its sums may be cut another way)
        assert rel_err(a[rid], b[rid]) < TOL8[dtype]


def _attention_plan(hd, window):
    """Order: attention, attention with a window, the first again with a cache of its own, a layer that reads the first's cache."""
    from gibbs_b200.config import ModelPlan, OrderEntry, PartSpec, prenorm_layer
    hidden, heads, kvh, vocab, eps = 128, 4, 2, 300, 1e-5
    norm = lambda name: PartSpec("rmsnorm", {"dim": hidden, "eps": eps}, {"weight": name})             # noqa: E731

    def attn(i, window=None, shares=False):
        t = {"q_proj.weight": f"l{i}.q", "out_proj.weight": f"l{i}.o", "q_norm.weight": f"l{i}.qn"}
        if not shares:
            t.update({"k_proj.weight": f"l{i}.k", "v_proj.weight": f"l{i}.v", "k_norm.weight": f"l{i}.kn"})
        return PartSpec("gqa_attention", {
            "hidden": hidden, "heads": heads, "kv_heads": kvh, "head_dim": hd, "bias": False, "qk_norm": True, "qk_norm_eps": eps,
            "scale": 1 / math.sqrt(hd), "window": window, "shares_kv": shares,
            "position": PartSpec("rope_half_split", {"head_dim": hd, "rotary_dim": hd, "theta": 1e4})}, t)

    ffn = lambda i: PartSpec("swiglu", {"hidden": hidden, "inner": 128, "bias": False},                # noqa: E731
                             {"gate.weight": f"l{i}.g", "up.weight": f"l{i}.u", "down.weight": f"l{i}.d"})
    mixers = [attn(0), attn(1, window=window), attn(2, shares=True)]
    layers = tuple(prenorm_layer(norm(f"l{i}.n1"), m, norm(f"l{i}.n2"), ffn(i)) for i, m in enumerate(mixers))
    order = (OrderEntry(0), OrderEntry(1), OrderEntry(0), OrderEntry(2, reads_cache_of=0))
    return ModelPlan("attention-only", vocab, hidden, 512, PartSpec("token_embedding", {"vocab": vocab, "dim": hidden}, {"weight": "emb"}),
                     layers, order, norm("fn"), PartSpec("lm_head", {"vocab": vocab, "dim": hidden}, {"weight": "emb"}))


def _plain_attention_model(w, ids, hd, window, heads=4, kvh=2, eps=1e-5):
    n, pos, inv = len(ids), torch.arange(len(ids)), plain.rope_inv_freq(hd, 1e4, torch.float64)
    x, first = w["emb"][torch.tensor(ids)], None
    for e, (i, reads) in enumerate([(0, None), (1, None), (0, None), (2, 0)]):
        h = plain.rms_norm(x, w[f"l{i}.n1"], eps)
        q = plain.rope_half_split(plain.rms_norm((h @ w[f"l{i}.q"].T).reshape(n, heads, hd), w[f"l{i}.qn"], eps), pos, inv)
        if reads is None:
            k = plain.rope_half_split(plain.rms_norm((h @ w[f"l{i}.k"].T).reshape(n, kvh, hd), w[f"l{i}.kn"], eps), pos, inv)
            v = (h @ w[f"l{i}.v"].T).reshape(n, kvh, hd)
            if e == 0:
                first = (k, v)
        else:
            k, v = first
        o = plain.causal_attention(q, k, v, 1 / math.sqrt(hd), window=window if i == 1 else None)
        x = x + o.reshape(n, heads * hd) @ w[f"l{i}.o"].T
        h = plain.rms_norm(x, w[f"l{i}.n2"], eps)
        g = h @ w[f"l{i}.g"].T
        x = x + (g / (1 + torch.exp(-g)) * (h @ w[f"l{i}.u"].T)) @ w[f"l{i}.d"].T
    return plain.rms_norm(x, w["fn"], eps) @ w["emb"].T


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd,window", [(64, 24), (16, 40)])
def test_windows_repeated_layers_and_shared_caches(oracle_in_8_bits, dtype, hd, window):
    from gibbs_b200.parts import build_model
    from gibbs_b200.weights import TensorDict, expected_tensors
    plan = _attention_plan(hd, window)
    torch.manual_seed(7)
    tensors = {}
    for name, decl in expected_tensors(plan).items():
        shape = decl.shapes[0]
        t = 1 + 0.1 * torch.randn(shape) if len(shape) == 1 else torch.randn(shape) * (0.3 if name == "emb" else 1.0 / math.sqrt(shape[-1]))
        tensors[name] = t.to(torch.bfloat16) if (dtype == "bfloat16" and len(shape) == 2) else t
    model = build_model(plan, TensorDict(tensors), torch.bfloat16 if dtype == "bfloat16" else torch.float32, DEV)
    w64 = {k: v.double() for k, v in tensors.items()}
    reqs = {f"r{i}": random_ids(80 + i, n, 300) for i, n in enumerate([70, 33, 100, 5])}
    want = {rid: _plain_attention_model(w64, ids, hd, window).numpy() for rid, ids in reqs.items()}
    for use_plan in (True, False):
        eng = _engine(model, n_pages={None: 40, window: 40}, use_plan=use_plan)
        assert (eng.plan is not None) == use_plan and len(eng.cache.groups) == 2
        for steps in (trace_whole(reqs), trace_portions(reqs), trace_mixed(reqs, capacity_tokens=320, seed=2)):
            got = run_trace_on_engine(eng, steps)
            for rid in reqs:
                bad = first_wrong(got[rid], want[rid], TOL8[dtype])
                assert bad is None, (use_plan, rid, bad)
        assert eng.cache.free_pages() == [40, 40]


def test_layers_that_do_not_take_8_bits_refuse():
    from gibbs_b200 import Engine
    from gibbs_b200.parts import build_model
    from gibbs_b200.weights import TensorDict, expected_tensors
    plan = _attention_plan(64, 24)
    layer = plan.layers[0]
    for role, category, spec in layer.parts:
        if role == "mixer":
            spec.params["softcap"] = 20.0
    torch.manual_seed(1)
    tensors = {n: torch.randn(d.shapes[0]) * 0.1 for n, d in expected_tensors(plan).items()}
    model = build_model(plan, TensorDict(tensors), torch.float32, DEV)
    with pytest.raises(ValueError, match="do not take"):
        Engine(model, n_pages={None: 8, 24: 8}, cache_dtype="float8_e4m3")
    with pytest.raises(ValueError, match="unknown cache dtype"):
        Engine(model, n_pages={None: 8, 24: 8}, cache_dtype="int4")
    Engine(model, n_pages={None: 8, 24: 8})


# ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("cache_dtype", [None, "float8_e4m3"])
@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("B", "bfloat16"), ("C", "bfloat16")])
@pytest.mark.parametrize("n", [1, 15, 16, 17, 70])
def test_a_forked_request_goes_on_like_one_that_ran_the_prompt(tmp_path_factory, name, dtype, n, cache_dtype):
    """Parent and child see the same logits while they get the same tokens, to the bit; with other tokens each goes its own way as
    a request of its own would, and neither disturbs the other."""
    from gibbs_b200 import StepEntry
    _, model = _model(tmp_path_factory, name, dtype)
    vocab = TINY[name][0]["vocab_size"]
    ids, more = random_ids(5, n, vocab), [random_ids(6 + i, 20, vocab) for i in range(3)]
    eng = _engine(model, cache_dtype=cache_dtype)
    eng.open("p")
    eng.step([StepEntry("p", ids, [n - 1])])
    eng.fork("p", "c")
    assert eng.length("c") == n
    logits = eng.step([StepEntry("p", [more[0][0]], [0]), StepEntry("c", [more[0][0]], [0])])
    assert torch.equal(logits[0], logits[1])
    eng.fork("c", "d")                                           # a fork of a fork, in the middle of a page or behind one
    got = {r: [] for r in "pcd"}
    for t in range(1, 20):
        rows = eng.step([StepEntry(r, [more[i][t]], [0]) for i, r in enumerate("pcd")]).cpu().numpy().copy()
        for i, r in enumerate("pcd"):
            got[r].append(rows[i])
        eng.check_status()
        eng.cache.check()
    eng.close("p")
    rows = eng.step([StepEntry("c", more[1][:7], list(range(7)))]).cpu().numpy()      # a portion, when the parent is gone
    got["c"] += list(rows)
    eng.check_status(), eng.cache.check()
    alone = _engine(model, cache_dtype=cache_dtype)
    for i, r in enumerate("pcd"):
        tail = [more[0][0]] + more[i][1:]
        full = ids + tail + (more[1][:7] if r == "c" else [])
        steps = [{"entries": [{"id": r, "tokens": ids + [tail[0]], "want": []}], "end": []}]
        steps += [{"entries": [{"id": r, "tokens": [t], "want": [0]}], "end": []} for t in tail[1:]]
        if r == "c":
            steps += [{"entries": [{"id": r, "tokens": more[1][:7], "want": list(range(7))}], "end": []}]
        steps[-1]["end"] = [r]
        want = run_trace_on_engine(alone, steps)[r]
        assert len(want) == len(got[r]) == len(full) - n - 1
        assert first_wrong(np.stack(got[r]), want, 2 * TOL8[dtype]) is None
    eng.close("c"), eng.close("d")
    assert eng.cache.free_pages() == [64]


def test_a_fork_that_finds_no_room_changes_nothing(tmp_path_factory):
    from gibbs_b200 import StepEntry
    from gibbs_b200.cache import OutOfPages, OutOfSlots, PoolError
    _, model = _model(tmp_path_factory, "A", "float32")
    eng = _engine(model, n_pages=2, max_requests=2)
    eng.open("p")
    eng.step([StepEntry("p", list(range(20)), [])])
    with pytest.raises(OutOfPages):
        eng.fork("p", "c")
    with pytest.raises(PoolError):
        eng.fork("x", "c")
    assert not eng.is_live("c")
    eng.step([StepEntry("p", list(range(12)), [])])              # 32 tokens: both pages are full
    eng.fork("p", "c")
    with pytest.raises(OutOfSlots):
        eng.fork("p", "d")
    eng.cache.check()


@pytest.mark.parametrize("dtype,cache_dtype", [("float32", None), ("float32", "float8_e4m3"), ("bfloat16", "float8_e4m3")])
def test_several_answers_to_a_prompt(tmp_path_factory, dtype, cache_dtype):
    from gibbs_b200 import Generator, SamplingParams
    folder, _ = _model(tmp_path_factory, "A", dtype)
    make = lambda: Generator(folder, dtype=dtype, device=DEV, ctx=256, page_size=PAGE, n_pages=64, max_running=4, cache_dtype=cache_dtype)  # noqa: E731
    prompt = random_ids(3, 37, TINY["A"][0]["vocab_size"])
    greedy = SamplingParams(temperature=0.0, max_new_tokens=12)
    gen = make()
    outs = gen.generate([prompt, prompt[:5]], greedy, stop_at_eos=False, samples=3)
    assert [len(o) for o in outs] == [3, 3] and all(a == o[0] and len(a) == 12 for o in outs for a in o)
    if dtype == "float32":
        assert outs[0][0] == make().generate([prompt], greedy, stop_at_eos=False)[0]
    drawn = SamplingParams(temperature=1.0, top_k=50, max_new_tokens=12, seed=9)
    got = gen.generate([prompt], drawn, stop_at_eos=False, samples=6)[0]             # more answers than places
    assert len(got) == 6 and len({tuple(a) for a in got}) > 1
    if dtype == "float32":
        each = [SamplingParams(temperature=1.0, top_k=50, max_new_tokens=12, seed=9 + i) for i in range(6)]
        assert got == make().generate([prompt] * 6, each, stop_at_eos=False)
    assert gen.engine.cache.free_pages() == [64]


# Each of two engines is within 2e-4 of its formulas in float32 (the bound of those designs' own tests).
@pytest.mark.parametrize("n", [13, 16, 61])
@pytest.mark.parametrize("name", ["A", "B", "C"])
@pytest.mark.parametrize("design", ["potivik", "petelix", "sisadra", "selivik", "guvetar", "nutopel"])
def test_forks_in_every_design(design, name, n):
    """State slots, latent rows, windows that keep a sequence's beginning, blocks of positions, tokens before: all go with a fork."""
    import importlib
    from gibbs_b200 import Engine, StepEntry
    h = importlib.import_module(design + "_helpers")
    cfg, seed = h.CONFIGS[name]
    key = (design, name)
    if key not in _models:
        _models[key] = h.build(name, "float32")[2] if design == "potivik" else h.build(cfg, seed, "float32")[1]
    make = lambda: Engine(_models[key], n_pages=96, page_size=16, max_requests=4, max_step_tokens=512, max_context=512, guard_cache=True)  # noqa: E731
    vocab = cfg["vocab"] if "vocab" in cfg else _models[key].vocab_size
    ids, tails = random_ids(1, n, vocab), [random_ids(2 + i, 24, vocab) for i in range(2)]
    tails[1][0] = tails[0][0]
    eng = make()
    eng.open("p")
    eng.step([StepEntry("p", ids, [n - 1])])
    eng.fork("p", "c")
    got = [[], []]
    for t in range(16):                                          # single tokens, beside each other
        rows = eng.step([StepEntry("p", [tails[0][t]], [0]), StepEntry("c", [tails[1][t]], [0])])
        assert t or torch.equal(rows[0], rows[1])
        for i in range(2):
            got[i].append(rows[i].cpu().numpy().copy())
    eng.close("p")
    got[1] += list(eng.step([StepEntry("c", tails[1][16:], list(range(8)))]).cpu().numpy())
    eng.check_status(), eng.cache.check()
    alone = make()
    for i, tail in enumerate(tails):
        tail = tail if i else tail[:16]
        steps = [{"entries": [{"id": "r", "tokens": ids, "want": []}], "end": []}]
        steps += [{"entries": [{"id": "r", "tokens": [t], "want": [0]}], "end": []} for t in tail[:16]]
        if i:
            steps += [{"entries": [{"id": "r", "tokens": tail[16:], "want": list(range(8))}], "end": []}]
        steps[-1]["end"] = ["r"]
        bad = first_wrong(np.stack(got[i]), run_trace_on_engine(alone, steps)["r"], 4e-4)
        assert bad is None, (i, bad)
    eng.close("c")
    assert eng.cache.free_pages() == [96] * len(eng.cache.groups)


@pytest.mark.parametrize("cache_dtype", [None, "float8_e4m3"])
@pytest.mark.parametrize("n", [20, 33, 80])
def test_forks_with_windows_and_shared_caches(n, cache_dtype):
    """A window gives shared pages back, one holder after the other, while both requests go on."""
    from gibbs_b200 import StepEntry
    from gibbs_b200.parts import build_model
    from gibbs_b200.weights import TensorDict, expected_tensors
    plan = _attention_plan(64, 24)
    torch.manual_seed(3)
    tensors = {}
    for name, decl in expected_tensors(plan).items():
        shape = decl.shapes[0]
        tensors[name] = 1 + 0.1 * torch.randn(shape) if len(shape) == 1 else torch.randn(shape) * (0.3 if name == "emb" else 1 / math.sqrt(shape[-1]))
    model = build_model(plan, TensorDict(tensors), torch.float32, DEV)
    ids, tails = random_ids(1, n, 300), [random_ids(2 + i, 40, 300) for i in range(2)]
    eng, alone = (_engine(model, n_pages={None: 40, 24: 40}, cache_dtype=cache_dtype) for _ in range(2))
    eng.open("p")
    eng.step([StepEntry("p", ids, [n - 1])])
    eng.fork("p", "c")
    got = [[], []]
    for t in range(40):
        rows = eng.step([StepEntry("p", [tails[0][t]], [0]), StepEntry("c", [tails[1][t]], [0])]).cpu().numpy()
        eng.check_status(), eng.cache.check()
        for i in range(2):
            got[i].append(rows[i].copy())
    eng.close("p"), eng.close("c")
    assert eng.cache.free_pages() == [40, 40]
    for i, tail in enumerate(tails):
        steps = [{"entries": [{"id": "r", "tokens": ids, "want": []}], "end": []}]
        steps += [{"entries": [{"id": "r", "tokens": [t], "want": [0]}], "end": []} for t in tail]
        steps[-1]["end"] = ["r"]
        assert first_wrong(np.stack(got[i]), run_trace_on_engine(alone, steps)["r"], 2 * TOL8["float32"]) is None
