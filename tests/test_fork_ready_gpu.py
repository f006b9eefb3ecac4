"""Forks load nothing and upload nothing that was not in place when the engine was made."""
import pytest
import torch

from helpers import make_folder, random_ids, TINY

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name,cache_dtype", [("A", None), ("C", None), ("A", "float8_e4m3")])
def test_the_first_fork_of_an_engine_finds_everything_in_place(tmp_path, monkeypatch, name, cache_dtype):
    from gibbs_b200 import Engine, StepEntry, load_model, ops
    model = load_model(make_folder(tmp_path, name, stored=torch.float32), dtype="float32", device="cuda:0")
    eng = Engine(model, n_pages=32, page_size=16, max_requests=4, max_step_tokens=128, cache_dtype=cache_dtype)
    tokens = random_ids(1, 21, TINY[name][0]["vocab_size"])
    eng.open("a")
    eng.step([StepEntry("a", tokens, [])])

    def not_now(*a, **k):
        raise AssertionError("a library is loaded, or a table made, by a fork")
    monkeypatch.setattr(ops.row_copies, "library", not_now)
    monkeypatch.setattr(ops, "RowCopies", not_now)
    eng.fork("a", "b")
    both = eng.step([StepEntry("a", [5], [0]), StepEntry("b", [5], [0])])
    assert torch.equal(both[0], both[1])


def test_a_cache_of_more_kinds_of_pages_than_a_fork_copies(tmp_path, monkeypatch):
    """An engine over it is made and steps as before; its forks are refused, and change nothing."""
    from gibbs_b200 import Engine, StepEntry, load_model, ops
    from gibbs_b200.engine.step import StepError
    model = load_model(make_folder(tmp_path, "A", stored=torch.float32), dtype="float32", device="cuda:0")
    monkeypatch.setattr(ops.row_copies, "MAX_GROUPS", 1)            # (pages and slots are two)
    eng = Engine(model, n_pages=32, page_size=16, max_requests=4, max_step_tokens=128)
    assert len(eng.cache.copied_tensors()) == 2
    eng.open("a")
    eng.step([StepEntry("a", [1, 2, 3], [])])
    with pytest.raises(StepError, match="fork"):
        eng.fork("a", "b")
    assert not eng.is_live("b") and eng.length("a") == 3
    eng.cache.check()
