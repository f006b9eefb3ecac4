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


@pytest.mark.parametrize("cache_dtype", [None, "float8_e4m3"])
@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("B", "bfloat16"), ("C", "bfloat16")])
def test_one_place_wanted_twice_beside_a_token_whose_logits_nobody_wants(tmp_path, name, dtype, cache_dtype):
    """As many tokens, requests and wanted rows as a decode step of that size has, but other rows: with graphs (which such a step then
    is recorded into, or replayed from) and without, before and after decode steps of that size."""
    from gibbs_b200 import Engine, StepEntry, load_model
    model = load_model(make_folder(tmp_path, name, stored=torch.bfloat16 if dtype == "bfloat16" else torch.float32), dtype=dtype, device="cuda:0")
    tokens = random_ids(2, 20, TINY[name][0]["vocab_size"])
    got = []
    for graphs in (False, True):
        eng = Engine(model, n_pages=32, page_size=16, max_requests=4, max_step_tokens=128, cache_dtype=cache_dtype, use_graphs=graphs)
        for r in "ab":
            eng.open(r)
        rows = [eng.step([StepEntry("a", tokens[:1], [0, 0]), StepEntry("b", tokens[1:2], [])]).clone()]
        rows.append(eng.step([StepEntry("a", tokens[2:3], [0]), StepEntry("b", tokens[3:4], [0])]).clone())
        rows.append(eng.step([StepEntry("a", tokens[4:5], []), StepEntry("b", tokens[5:6], [0, 0])]).clone())
        rows.append(eng.step([StepEntry("a", tokens[6:7], [0]), StepEntry("b", tokens[7:8], [0])]).clone())
        eng.fork("b", "c")
        rows.append(eng.step([StepEntry("c", tokens[8:9], [0]), StepEntry("b", tokens[8:9], [0])]).clone())
        eng.check_status()
        assert torch.equal(rows[0][0], rows[0][1]) and torch.equal(rows[2][0], rows[2][1]) and torch.equal(rows[4][0], rows[4][1])
        assert not torch.equal(rows[1][0], rows[1][1])
        got.append(rows)
    assert all(torch.equal(a, b) for a, b in zip(*got))
