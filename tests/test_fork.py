"""Forked requests and several answers to one prompt, as far as it needs no GPU: pages and slots in the manager, the scheduler on
a fake engine that forks."""
import numpy as np
import pytest
import torch

from fake_engine import FakeEngine, fake_next
from gibbs_b200 import SamplingParams
from gibbs_b200.cache import CacheManager, IdPool, OutOfPages, OutOfSlots, PoolError
from gibbs_b200.engine.scheduler import FinishReason, Scheduler
from gibbs_b200.parts.base import PagedKV, PagedRows, SlotState

F8 = torch.float8_e4m3fn


def test_an_id_has_as_many_holders_as_it_was_given():
    p = IdPool(2, "page")
    a = p.take()
    assert p.share(a) == a and p.holders(a) == 2 and p.n_shared == 1 and p.n_used == 1
    p.give_back(a)
    assert p.holders(a) == 1 and p.n_shared == 0 and p.n_free == 1
    p.check()
    p.give_back(a)
    assert p.n_free == 2
    with pytest.raises(PoolError):
        p.give_back(a)
    with pytest.raises(PoolError):
        p.share(a)
    with pytest.raises(PoolError):
        p.share(5)


def _manager(n_pages=12, page=4, slots=4, window=None, state=True):
    needs = [([PagedKV(2, 4)], None), ([PagedKV(1, 8, window)], None), ([PagedRows(3)], None)]
    if state:
        needs.append(([SlotState((5,))], None))
    return CacheManager(needs, n_pages, page, slots, torch.float32, "cpu", 200)


def _grow(m, rc, n):
    m.reserve(rc, rc.length + n)
    m.advance(rc, rc.length + n)


@pytest.mark.parametrize("length", [0, 1, 3, 4, 5, 8, 11])
def test_full_pages_are_shared_and_the_last_one_is_copied(length):
    m = _manager()
    a = m.open("a")
    if length:
        _grow(m, a, length)
    before = m.free_pages()
    pairs = m.fork("a", "b")
    b = m.live["b"]
    assert b.length == length and len(pairs) == len(m.groups) + 1 and pairs[-1] == [(a.slot, b.slot)]
    full = length // 4
    for g in range(len(m.groups)):
        assert b.block_tables[g][:full] == a.block_tables[g][:full]
        if length % 4:
            assert pairs[g] == [(a.block_tables[g][full], b.block_tables[g][full])] and pairs[g][0][0] != pairs[g][0][1]
            assert m.free_pages()[g] == before[g] - 1
        else:
            assert pairs[g] == [] and m.free_pages()[g] == before[g]
    m.check()
    _grow(m, a, 6), _grow(m, b, 9)
    m.check()
    m.close("a")
    m.check()
    _grow(m, b, 1)
    m.close("b")
    m.check()
    assert m.free_pages() == [12] * len(m.groups) and m.slots.n_free == 4


def test_fork_takes_nothing_when_it_cannot():
    m = _manager(n_pages=2, slots=3)
    a = m.open("a")
    _grow(m, a, 7)
    with pytest.raises(OutOfPages):
        m.fork("a", "b")
    assert list(m.live) == ["a"] and m.slots.n_free == 2 and m.free_pages() == [0] * len(m.groups)
    _grow(m, a, 1)                                              # (the page is full now and can be shared)
    m.fork("a", "b"), m.fork("b", "c")
    with pytest.raises(OutOfSlots):
        m.fork("a", "d")
    with pytest.raises(PoolError):
        m.fork("a", "b")
    with pytest.raises(PoolError):
        m.fork("x", "e")
    assert m.groups[0].pool.holders(a.block_tables[0][0]) == 3
    m.check()


def test_a_window_gives_back_a_shared_page_with_its_last_holder():
    m = CacheManager([([PagedKV(1, 4, 6)], None)], 6, 4, 4, torch.float32, "cpu", 400)
    a = m.open("a")
    _grow(m, a, 8)
    m.fork("a", "b")
    b = m.live["b"]
    first = a.block_tables[0][0]
    # positions 8..13 pass the first page (positions 0..3 have left the window of 6 from 9 on)
    assert m.pages_wanted([(a, 12)]) == [1] and m.pages_wanted([(a, 12), (b, 12)]) == [2]
    _grow(m, a, 4), _grow(m, b, 4)
    assert m.pages_wanted([(a, 16)]) == [1]                     # (b holds it still)
    assert m.pages_wanted([(a, 16), (b, 16)]) == [1]            # one page falls free for the two taken
    assert m.free_pages() == [2]
    m.reserve_all([(a, 16), (b, 16)])
    assert a.block_tables[0][0] == -1 and b.block_tables[0][0] == -1 and m.groups[0].pool.holders(first) in (0, 1)
    m.advance(a, 16), m.advance(b, 16)
    m.check()


@pytest.mark.parametrize("seed", range(4))
def test_random_orders_of_requests_and_forks(seed):
    rng = np.random.default_rng(seed)
    m = _manager(n_pages=14, slots=5, window=None if seed % 2 else 9, state=seed < 2)
    live, n = {}, 0
    for _ in range(500):
        r = rng.random()
        if r < 0.15 and len(live) < 5:
            live[n] = m.open(n)
            n += 1
        elif r < 0.35 and live and len(live) < 5:
            parent = int(rng.choice(list(live)))
            before = (m.free_pages(), m.slots.n_free)
            try:
                m.fork(parent, n)
                live[n] = m.live[n]
                n += 1
            except OutOfPages:
                assert before == (m.free_pages(), m.slots.n_free)
        elif r < 0.8 and live:
            rc = live[int(rng.choice(list(live)))]
            grow = int(rng.integers(1, 8))
            if rc.length + grow <= 100 and m.can_reserve(rc, rc.length + grow):
                _grow(m, rc, grow)
        elif r < 0.87 and len(live) > 1:
            wants = [(rc, rc.length + 1) for rc in live.values()]
            if m.can_reserve_all(wants):
                m.reserve_all(wants)
                if rng.random() < 0.5:
                    for rc, _ in wants:
                        m.unreserve(rc)
                else:
                    for rc, to in wants:
                        m.advance(rc, to)
        elif live:
            i = int(rng.choice(list(live)))
            m.close(i)
            del live[i]
        m.check()
    for i in list(live):
        m.close(i)
    m.check()
    assert all(f == g.pool.size for f, g in zip(m.free_pages(), m.groups))


def test_an_8_bit_cache_in_the_manager():
    needs = [([PagedKV(2, 16, in_8_bits=True)], None), ([SlotState((2,))], None), ([], 0)]
    m = CacheManager(needs, 6, 4, 2, torch.bfloat16, "cpu", 64, guard=True, kv_dtype=F8)
    assert m.kv_bytes_per_token() == 2 * 2 * 16
    views = m.views([torch.zeros(1, m.max_blocks, dtype=torch.int32)], torch.zeros(1, dtype=torch.int32), [0])
    p = views[0][0].in_8_bits
    assert p.k is views[0][0].k_pages and p.k.dtype == F8 and p.k_scales.shape == (6, 2) and views[2][0].in_8_bits is p
    assert [len(t) for t in m.copied_tensors()] == [4, 1]
    m.check()
    p.v_scales.as_strided((1,), (1,), p.v_scales.storage_offset() + p.v_scales.numel())[0] = 9.0
    with pytest.raises(PoolError, match="guard"):
        m.check()
    with pytest.raises(ValueError, match="do not take"):
        CacheManager([([PagedKV(2, 16)], None)], 6, 4, 2, torch.bfloat16, "cpu", 64, kv_dtype=F8)
    with pytest.raises(ValueError, match="no layer"):
        CacheManager([([PagedRows(16)], None)], 6, 4, 2, torch.bfloat16, "cpu", 64, kv_dtype=F8)
    with pytest.raises(ValueError, match="held in"):
        CacheManager(needs, 6, 4, 2, torch.bfloat16, "cpu", 64, kv_dtype=torch.float16)
    assert CacheManager(needs, 6, 4, 2, torch.bfloat16, "cpu", 64, kv_dtype=torch.bfloat16).in_8_bits is False


def test_cache_dtypes_by_name():
    from gibbs_b200.engine.step import parse_cache_dtype
    assert parse_cache_dtype(None) is None and parse_cache_dtype("float8_e4m3") == F8 and parse_cache_dtype(F8) == F8
    for bad in ("int4", torch.float16, torch.bfloat16):
        with pytest.raises(ValueError):
            parse_cache_dtype(bad)


# ---------------------------------------------------------------------------------------------------
class ForkingEngine(FakeEngine):
    """The fake engine with a fork: what a request was fed goes along."""
    max_step_tokens = 64

    def fork(self, parent, child):
        self.cache.fork(parent, child)
        self.fed[child] = list(self.fed[parent])
        self.events.append("fork")


class SeededSampler:
    """Picks by the logits (fake: one-hot) and the request's seed and count, and may lag like the real one."""

    def __init__(self, vocab):
        self.vocab, self.rows = vocab, []

    def __call__(self, logits, params, seeds, counters, recent=None):
        best = [int(i) for i in logits.argmax(-1)]
        assert len(best) == len(params) == len(seeds) == len(counters)
        self.rows.append(len(best))
        return [(b + 7 * s + 3 * c) % self.vocab for b, s, c in zip(best, seeds, counters)]

    def sample_async(self, logits, params, seeds, counters, recent=None):
        picked = self(logits, params, seeds, counters)

        class Pending:
            device_ids = torch.tensor(picked, dtype=torch.int32)

            def wait(self):
                return picked
        return Pending()


def _answers(engine, prompt, n, params, samples=True, **k):
    sched = Scheduler(engine, SeededSampler(engine.vocab), **k)
    if samples:
        ids = sched.submit(prompt, params, samples=n)
    else:
        ids = [sched.submit(prompt, SamplingParams(**{**params.__dict__, "seed": params.seed + i})) for i in range(n)]
    outs = sched.run(max_steps=2000)
    assert not sched.has_work()
    engine.cache.check()
    assert all(f == g.pool.size for f, g in zip(engine.cache.free_pages(), engine.cache.groups))
    return [list(sched.sequences[i].output) for i in ids], sched, outs


@pytest.mark.parametrize("overlap", [False, True])
@pytest.mark.parametrize("prompt_len,n,budget", [(1, 3, 64), (5, 4, 64), (9, 4, 3), (16, 2, 64)])
def test_answers_equal_those_of_requests_of_their_own(overlap, prompt_len, n, budget):
    params = SamplingParams(max_new_tokens=9, seed=11)
    prompt = list(range(1, prompt_len + 1))
    want, _, _ = _answers(FakeEngine(), prompt, n, params, samples=False)
    eng = ForkingEngine()
    got, _, _ = _answers(eng, prompt, n, params, overlap=overlap, max_batch_tokens=budget)
    assert got == want and eng.events.count("fork") == n - 1
    # the prompt was run once
    assert sum(k for step in eng.log if step != "failed" for _, k, _ in [(e[0], e[1], e[2]) for e in step] if k > 1) in (0, prompt_len) or budget == 3
    assert len({tuple(g) for g in got}) == n


def test_more_answers_than_places():
    """Six answers on four places, and on pages for two: the rest run later; answers do not change."""
    params = SamplingParams(max_new_tokens=6, seed=3)
    want, _, _ = _answers(FakeEngine(max_requests=4), [5, 6, 7], 6, params, samples=False)
    for eng in (ForkingEngine(max_requests=4), ForkingEngine(max_requests=4, n_pages=6), ForkingEngine(max_requests=1)):
        got, _, _ = _answers(eng, [5, 6, 7], 6, params)
        assert got == want
    eng = FakeEngine(max_requests=4)                            # an engine that cannot fork
    assert _answers(eng, [5, 6, 7], 6, params)[0] == want
    eng = ForkingEngine(max_requests=4)
    eng.max_step_tokens = 4                                     # room for fewer rows of logits than answers
    assert _answers(eng, [5, 6, 7], 6, params, max_batch_tokens=4)[0] == want


def test_a_leader_that_ends_early_leaves_its_prompt_to_the_next():
    params = SamplingParams(max_new_tokens=5, seed=1)
    want, _, _ = _answers(FakeEngine(), [4, 5, 6, 7, 8], 3, params, samples=False)
    for when in (0, 1):
        eng = ForkingEngine()
        sched = Scheduler(eng, SeededSampler(eng.vocab), max_batch_tokens=2)
        ids = sched.submit([4, 5, 6, 7, 8], params, samples=3)
        for _ in range(when):
            sched.step()
        sched.cancel(ids[0])
        sched.run(max_steps=200)
        assert sched.sequences[ids[0]].finish == FinishReason.CANCELLED
        assert [sched.sequences[i].output for i in ids[1:]] == want[1:]
        eng.cache.check()
    # a follower that gives up while it waits
    eng = ForkingEngine()
    sched = Scheduler(eng, SeededSampler(eng.vocab), max_batch_tokens=2)
    ids = sched.submit([4, 5, 6, 7, 8], params, samples=3)
    sched.step()
    sched.cancel(ids[1])
    sched.run(max_steps=200)
    assert [sched.sequences[i].finish for i in ids] == [FinishReason.LENGTH, FinishReason.CANCELLED, FinishReason.LENGTH]
    assert sched.sequences[ids[0]].output == want[0] and sched.sequences[ids[2]].output == want[2]
    # a step that fails ends the request that runs the prompt; the others run it again
    eng = ForkingEngine(fail_on=0)
    sched = Scheduler(eng, SeededSampler(eng.vocab))
    ids = sched.submit([4, 5, 6, 7, 8], params, samples=3)
    sched.run(max_steps=200)
    assert sched.sequences[ids[0]].finish == FinishReason.ERROR
    assert [sched.sequences[i].output for i in ids[1:]] == want[1:]


def test_zero_new_tokens_and_refusals():
    eng = ForkingEngine()
    got, sched, _ = _answers(eng, [1, 2], 3, SamplingParams(max_new_tokens=0, seed=0))
    assert got == [[], [], []] and all(s.finish == FinishReason.LENGTH for s in sched.sequences.values())
    with pytest.raises(ValueError):
        sched.submit([1], samples=0)
    sched = Scheduler(ForkingEngine(), SeededSampler(50))
    outs = sched.generate([[1, 2, 3], [4]], SamplingParams(max_new_tokens=4, seed=2), samples=2)
    assert [len(o) for o in outs] == [2, 2] and all(len(a) == 4 for o in outs for a in o)
    assert isinstance(fake_next([1], 50), int)
