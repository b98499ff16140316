"""CPU: the work space of attention is asked for on the pool's device, whose SMs decide how keys are split, whichever device is the current one."""
import contextlib
from types import SimpleNamespace

import pytest
import torch

import lit_llama_b200.paged as paged
from lit_llama_b200 import PagedCache, PagedStep


@pytest.mark.parametrize("tree", [False, True])
def test_work_spaces_are_those_of_the_pools_device(tree, monkeypatch):
    current, asked = [0], []

    @contextlib.contextmanager
    def device(d):
        before, index = current[0], d.index if isinstance(d, torch.device) else d
        current[0] = index if index >= 0 else before
        yield
        current[0] = before

    def work(*sizes):
        asked.append(current[0])
        return 100 + current[0]

    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(paged.S, "lib", lambda: SimpleNamespace(b2l_seq_paged_attention_work=work, b2l_seq_paged_attention_tree_work=work))
    cache, step = PagedCache.empty(4, 16, 2, 32, device="cpu"), PagedStep.of([(2, 2, [0])], torch.device("cpu"))
    for at, floats in ((torch.device("cuda", 1), 101), (torch.device("cpu"), 100)):
        monkeypatch.setattr(cache, "device", at)
        assert cache._plan(2, 4, None, 0, 0, step, tree)[0] == floats
    assert asked == [1, 0] and current == [0]
