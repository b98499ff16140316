"""GPU: what the attention of trees, acceptance and selection give is the same, bit by bit, from call to call."""
import random

import pytest
import torch

from test_gpu_tree import BF, F32, flat, setup, steered, trees_of

pytestmark = pytest.mark.gpu

SEQUENCES = [(32, 700), (1, 300), (30, 1290), (17, 129), (3, 3), (25, 2000)]


@pytest.mark.parametrize("form,store,dtype", [("joined", "act", BF), ("few", "act", F32), ("few", "fp8", BF), ("pair", "act", BF), ("pair", "fp8", BF), ("pair", "int8", BF), ("many", "act", BF),
                                              ("many", "fp8", BF), ("many", "int8", BF)], ids=str)
def test_attention_repeats_itself(form, store, dtype):
    from lit_llama_b200 import PagedTree

    cache, q, step, seqs = setup(SEQUENCES if form != "joined" else SEQUENCES[:1], 16, 2, 8, 128, 128, store, dtype)
    if form != "joined":
        step = steered(seqs, 4, form)
    tree = PagedTree(step, flat(trees_of(seqs, random.Random(3))), nodes=32)
    once = cache.attend(q, step, tree=tree)
    assert all(torch.equal(cache.attend(q, step, tree=tree), once) for _ in range(50))
