"""Steps of trees of drafted tokens on the host: what a session may still accept, and which pages it holds, when steps are
refused, fail, or go on without accepting."""

import pytest
import torch

from ninfer_amd_mi50_b200.cache import CacheManager, OutOfPages
from ninfer_amd_mi50_b200.engine import BatchError, ModelRunner, StepEntry, TreeEntry
from ninfer_amd_mi50_b200.parts.base import CacheSpec

PAGE = 4


class Model:
    """Says nothing of interest; `fails` makes the next pass raise."""
    vocab_size, graph_safe, tree_safe, fails = 50, False, True, False

    def forward(self, ctx, cache_view, state_of):
        if self.fails:
            raise RuntimeError("no pass")
        return torch.zeros(len(ctx.logit_rows), self.vocab_size)


@pytest.fixture
def runner():
    cache = CacheManager([CacheSpec("full", 1, 16)], [None], page_size=PAGE, num_pages=8, max_requests=3, max_context=64)
    return ModelRunner(Model(), cache, torch.float32, "cpu")


def start(runner, req, length):
    runner.open(req)
    runner.step([StepEntry(req, [1] * length)])


def free(runner):
    runner.cache.check()
    return runner.cache.pages_free()[0]


@pytest.mark.parametrize("then", ["step", "tree"])
@pytest.mark.parametrize("own", [False, True], ids=["another's", "its own"])
def test_a_refused_step_leaves_trees_to_be_accepted(runner, then, own):
    start(runner, "a", 6)
    start(runner, "b", 5)
    runner.tree_step([TreeEntry("a", [1] * 7)])              # 13 places: 4 of 8 pages, "b" has 2
    assert free(runner) == 2
    too_many = "a" if own else "b"
    for order in (("a", "b"), ("b", "a")):
        sizes = {"a": 1, "b": 1, too_many: 30}
        with pytest.raises(OutOfPages):
            if then == "step":
                runner.step([StepEntry(r, [1] * sizes[r]) for r in order])
            else:
                runner.tree_step([TreeEntry(r, [1] * sizes[r]) for r in order])
        assert free(runner) == 2 and runner.cache.length("a") == 6
    runner.accept({"a": [1, 2, 3]})
    assert runner.cache.length("a") == 10 and free(runner) == 3
    with pytest.raises(BatchError):
        runner.accept({"a": [1]})


def test_a_refused_step_takes_pages_back(runner):
    start(runner, "a", 4)
    start(runner, "b", 4)
    with pytest.raises(OutOfPages):
        runner.step([StepEntry("a", [1] * 8), StepEntry("b", [1] * 30)])
    assert free(runner) == 6
    with pytest.raises(OutOfPages):
        runner.tree_step([TreeEntry("a", [1] * 8), TreeEntry("b", [1] * 30)])
    assert free(runner) == 6 and not runner.trees


def test_a_pass_that_fails_ends_trees(runner):
    """Rows of theirs may have been written over."""
    start(runner, "a", 6)
    runner.tree_step([TreeEntry("a", [1] * 7)])
    runner.model.fails = True
    for step in (lambda: runner.step([StepEntry("a", [1])]), lambda: runner.tree_step([TreeEntry("a", [1, 2])])):
        with pytest.raises(RuntimeError, match="no pass"):
            step()
        assert free(runner) == 6
        with pytest.raises(BatchError):
            runner.accept({"a": [1]})


def test_pages_of_a_tree_that_was_not_accepted_are_given_back(runner):
    """With the step that writes over it, not at the session's end."""
    start(runner, "a", 6)
    runner.tree_step([TreeEntry("a", [1] * 20)])             # 26 places: 7 pages
    assert free(runner) == 1
    runner.step([StepEntry("a", [1])])
    assert free(runner) == 6
    runner.tree_step([TreeEntry("a", [1] * 20)])
    runner.tree_step([TreeEntry("a", [1, 2])])
    assert free(runner) == 5
    runner.accept({"a": [1]})
    assert runner.cache.length("a") == 9 and free(runner) == 5
