"""Several answers to a prompt where forks raise."""
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
