"""Several answers to a prompt where forks raise, and where a client goes while it waits."""
import pytest

from fake_engine import FakeEngine
from gibbs_b200 import SamplingParams
from gibbs_b200.engine.scheduler import FinishReason, Scheduler
from test_fork import ForkingEngine, SeededSampler, _answers


class FailingForks(ForkingEngine):
    """Raises at the forks of the given numbers, before anything is taken."""

    def __init__(self, fails, **k):
        super().__init__(**k)
        self.fails, self.forks = fails, 0

    def fork(self, parent, child):
        self.forks += 1
        if self.forks - 1 in self.fails:
            raise RuntimeError("no such library")
        super().fork(parent, child)


@pytest.mark.parametrize("overlap", [False, True])
@pytest.mark.parametrize("fails", [{0}, {1}, {0, 1, 2}, set(range(100))])
def test_a_fork_that_raises_leaves_its_prompt_to_be_run_again(fails, overlap):
    """Nobody's token is lost, and the requests that were not forked run the prompt themselves."""
    params = SamplingParams(max_new_tokens=6, seed=3)
    prompt = [5, 6, 7, 8, 9]
    want, _, _ = _answers(FakeEngine(), prompt, 4, params, samples=False)
    eng = FailingForks(fails)
    with pytest.warns(RuntimeWarning, match="no such library"):
        got, sched, outs = _answers(eng, prompt, 4, params, overlap=overlap)
    assert got == want and eng.forks >= 3
    assert all(s.finish == FinishReason.LENGTH for s in sched.sequences.values())
    assert sum(len(o.emitted) for o in outs) == 24


@pytest.mark.filterwarnings("ignore:a fork failed")
def test_a_fork_that_raises_beside_other_requests():
    """The tokens of the other requests of that step are emitted."""
    eng = FailingForks(set(range(100)))
    sched = Scheduler(eng, SeededSampler(eng.vocab))
    other = sched.submit([1, 2], SamplingParams(max_new_tokens=8, seed=0))
    sched.step()
    ids = sched.submit([4, 5, 6], SamplingParams(max_new_tokens=3, seed=1), samples=2)
    with pytest.warns(RuntimeWarning):
        out = sched.step()
    assert {i for i, _ in out.emitted} == {other, ids[0]}
    sched.run(max_steps=200)
    assert not sched.has_work() and [len(sched.sequences[i].output) for i in [other] + ids] == [8, 3, 3]
    eng.cache.check()


# ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("overlap", [False, True])
def test_an_answer_that_waits_for_its_prompt_ends_at_the_step_after_its_cancellation(overlap):
    """Wherever the request that runs the prompt is: running it, or waiting for a place behind another request."""
    params = SamplingParams(max_new_tokens=5, seed=1)
    want, _, _ = _answers(FakeEngine(), [4, 5, 6, 7, 8], 3, params, samples=False)
    for places, before in ((8, 0), (8, 1), (1, 0), (1, 2)):
        eng = ForkingEngine()
        sched = Scheduler(eng, SeededSampler(eng.vocab), max_batch_tokens=2, max_running=places, overlap=overlap)
        if places == 1:
            sched.submit([1], SamplingParams(max_new_tokens=12, seed=0))
        ids = sched.submit([4, 5, 6, 7, 8], params, samples=3)
        for _ in range(before):
            sched.step()
        sched.cancel(ids[1])
        out = sched.step()
        assert (ids[1], FinishReason.CANCELLED) in out.finished
        assert sched.sequences[ids[1]].finish == FinishReason.CANCELLED
        sched.cancel(ids[1])                                       # (again: nothing)
        outs = sched.run(max_steps=300)
        assert not sched.has_work() and all(i != ids[1] for o in outs for i, _ in o.finished + o.emitted)
        assert [sched.sequences[i].output for i in ids] == [want[0], [], want[2]]
        eng.cache.check()


def test_an_answer_that_was_cancelled_takes_no_row_of_logits():
    """Two of five answers are cancelled between the steps of a prompt; the engine has room for three rows beside the first's."""
    eng = ForkingEngine()
    eng.max_step_tokens = 3
    sampler = SeededSampler(eng.vocab)
    sched = Scheduler(eng, sampler, max_batch_tokens=3)
    ids = sched.submit([4, 5, 6, 7, 8], SamplingParams(max_new_tokens=4, seed=1), samples=5)
    sched.step()
    sched.cancel(ids[1]), sched.cancel(ids[2])
    sched.step()                                                   # (the prompt's last tokens)
    assert sampler.rows[-1] == 3 and eng.events.count("fork") == 2
    sched.run(max_steps=100)
    assert [len(sched.sequences[i].output) for i in ids] == [4, 0, 0, 4, 4]


def test_all_that_wait_are_cancelled_or_the_leader_with_one_of_them():
    for gone in ((1, 2), (0, 1), (0, 1, 2)):
        eng = ForkingEngine()
        sched = Scheduler(eng, SeededSampler(eng.vocab), max_batch_tokens=2)
        ids = sched.submit([4, 5, 6, 7, 8], SamplingParams(max_new_tokens=4, seed=1), samples=3)
        sched.step()
        for i in gone:
            sched.cancel(ids[i])
        out = sched.step()
        assert sorted(i for i, _ in out.finished) == sorted(ids[i] for i in gone)
        sched.run(max_steps=100)
        assert not sched.has_work()
        assert [sched.sequences[i].finish for i in ids] == [FinishReason.CANCELLED if i in gone else FinishReason.LENGTH for i in range(3)]
        assert all(f == g.pool.size for f, g in zip(eng.cache.free_pages(), eng.cache.groups))


def test_a_prompt_given_as_an_iterator():
    """(As for one answer: the prompt is gone through once.)"""
    params = SamplingParams(max_new_tokens=4, seed=1)
    want, _, _ = _answers(ForkingEngine(), [4, 5, 6, 7, 8], 3, params)
    assert _answers(ForkingEngine(), iter([4, 5, 6, 7, 8]), 3, params)[0] == want


def test_a_prompt_that_is_refused_leaves_nothing_behind():
    eng = ForkingEngine()
    sched = Scheduler(eng, SeededSampler(eng.vocab))
    with pytest.raises(ValueError):
        sched.submit([1] * (eng.max_context + 1), SamplingParams(seed=0), samples=3)
    assert not sched.has_work() and not sched.sequences
