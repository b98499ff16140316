"""CPU: how many new tokens the masks of a tree have room for: as many as a sequence has, never what a hint says."""
import pytest
import torch

import lit_llama_b200.paged as paged
from lit_llama_b200 import PagedStep, PagedTree

CPU = torch.device("cpu")


@pytest.fixture(autouse=True)
def no_launches(monkeypatch):
    monkeypatch.setattr(paged, "_launch", lambda *a: None)


def chain(n):
    return torch.arange(-1, n - 1, dtype=torch.int32)


def of(*news):
    return PagedStep.of([(n, n + 5, [0]) for n in news], CPU)


@pytest.mark.parametrize("hint", [0, 1, 4, 64])
def test_a_hint_does_not_decide(hint):
    made = of(63, 1)
    step = PagedStep(made.starts.clone(), made.lengths, made.table, rows=64, max_new=hint)
    assert PagedTree(step, chain(64)).words == 2
    assert PagedTree(made, chain(64)).words == 2 and PagedTree(of(32, 32), chain(64)).words == 1
    assert PagedTree(step, chain(64), nodes=20).words == 1 and PagedTree(PagedStep.of([], CPU), chain(0)).words == 1


def test_a_step_that_is_refilled():
    step = of(32, 32)
    tree = PagedTree(step, chain(64))
    before = step.starts.clone()
    for other in (of(63, 1), of(33, 31)):
        with pytest.raises(ValueError, match="nodes"):
            step.refill(other)
        assert torch.equal(step.starts, before)
    step.refill(of(32, 32))
    wide = of(32, 32)
    trees = [PagedTree(wide, chain(64), nodes=64), tree]
    wide.refill(of(63, 1))
    assert wide.starts.tolist() == [0, 63, 64] and PagedTree(wide, chain(64)).words == 2
    unknown = PagedStep(before, step.lengths, step.table, rows=64, max_new=32)      # of tensors: any of its rows may be one sequence's
    with pytest.raises(ValueError, match="nodes"):
        step.refill(unknown)
    wide.refill(unknown)
    del tree, trees
    step.refill(of(63, 1))                                                 # nobody has masks of it any more


def test_a_step_that_is_written_over():
    step, other = of(32, 32), of(32, 32)
    tree = PagedTree(step, chain(64))
    for s in (step, other):                                                # longer sequences, other pages: as many new tokens
        s.lengths.add_(1)
        s.table.fill_(1)
        assert PagedTree(s, chain(64)).words == 1
    step.refill(other)
    assert step.lengths.tolist() == [38, 38] and tree.words == 1
    step.starts.copy_(torch.tensor([0, 63, 64], dtype=torch.int32))
    assert PagedTree(step, chain(64)).words == 2
    with torch.inference_mode():
        assert PagedTree(of(32, 32), chain(64)).words == 1
