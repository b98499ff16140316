"""GPU: rows of trees that are computed again, as a value that they do not see is infinite: what they see is what their masks say, whatever the window."""
import pytest
import torch

import tree_oracle as T
from test_gpu_tree import BF, DEV, F32, check, flat, setup, sights, steered

pytestmark = pytest.mark.gpu

FORMS = [("joined", "act", BF), ("joined", "act", F32), ("joined", "int8", BF), ("few", "act", BF), ("few", "fp8", BF), ("few", "act", F32), ("pair", "act", BF), ("pair", "fp8", BF),
         ("many", "act", BF), ("many", "int8", BF)]


def again(parents, base, form, store, dtype, window, first, own):
    """The tree `parents` over `base` tokens; its last token, which follows the sequence and nobody else sees, is infinite.  `own`: whether the masks have the window too."""
    from lit_llama_b200 import PagedStep, PagedTree

    n = len(parents)
    cache, q, step, seqs = setup([(n, base + n)], 16, 2, 2, 64, 64, store, dtype)
    whole = PagedStep.of([(base + n, base + n, seqs[0][2])], DEV)
    k, v = cache.read(whole)
    v[-1] = float("inf")
    cache.write(k, v, whole)                                               # 8-bit rows are quantised again: the oracle reads what is there now
    if form != "joined":
        step = steered(seqs, 1, form)
    tree = PagedTree(step, flat([parents]), nodes=n, window=window if own else 0, first=first if own else 0)
    sets, depths = sights(seqs, [parents], window if own else 0, first if own else 0)
    got = cache.attend(q, step, tree=tree, window=window, first=first)
    assert n - 1 in sets[-1] and not any(n - 1 in s for s in sets[:-1]) and not torch.isfinite(got[-1]).any()
    want = T.attend(q, cache, seqs, sets[:-1] + [set()], depths, 64 ** -0.5, window, first)
    check(got[:-1], tuple(x[:-1] for x in want), 64, base + n, dtype == F32, store)


@pytest.mark.parametrize("form,store,dtype", FORMS, ids=str)
@pytest.mark.parametrize("window,first", [(16, 0), (1, 0), (40, 70)])
def test_masks_without_a_window_under_a_window(window, first, form, store, dtype):
    """A chain of 96: the last of them see 96 new tokens, more than the window has."""
    again([i - 1 for i in range(96)] + [-1], 200, form, store, dtype, window, first, False)


@pytest.mark.parametrize("form,store,dtype", FORMS, ids=str)
def test_a_first_position_at_a_later_place(form, store, dtype):
    """A branch of 71 tokens behind a chain of 40: its first ones are at positions below `first`, their keys at places above it."""
    again([i - 1 for i in range(40)] + [5] + list(range(40, 110)) + [-1], 200, form, store, dtype, 4, 220, True)


@pytest.mark.parametrize("hint", [0, 1, 16, 70])
@pytest.mark.parametrize("store", ["act", "fp8"])
def test_hints_do_not_hide_tokens(store, hint):
    """A step of tensors whose longest sequence is not what the host says."""
    from lit_llama_b200 import PagedStep, PagedTree

    cache, q, step, seqs = setup([(70, 170), (3, 20)], 16, 1, 4, 64, 64, store, BF)
    step = PagedStep(step.starts, step.lengths, step.table, rows=step.rows, max_new=hint)
    trees = [[i - 1 for i in range(70)], [-1, 0, 0]]
    sets, depths = sights(seqs, trees)
    check(cache.attend(q, step, tree=PagedTree(step, flat(trees))), T.attend(q, cache, seqs, sets, depths, 64 ** -0.5), 64, 170, False, store)


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("temperature", [1e-39, 2e-38, 1.0])
def test_drawn_targets_where_quotients_and_noise_are_infinite(temperature, dtype):
    """Noise of 0 (its token wins, whatever its logit) and of infinity (it never does), at temperatures whose reciprocal f32 does not have."""
    from lit_llama_b200 import PagedStep, PagedTree

    g = torch.Generator().manual_seed(5)
    x = torch.randn(12, 9000, generator=g).to(dtype)
    noise = torch.empty(12, 9000).exponential_(generator=g)
    noise[0, 700], noise[1, 8999], noise[2, 5], noise[2, 8500], noise[3, :] = 0.0, 0.0, 0.0, 0.0, float("inf")
    x[0, 700], x[1, 8999], x[2, 5], x[2, 8500] = -9.0, 9.0, -1.0, 2.0
    x[4, :], x[5, ::2], x[6, 77] = 0.0, -0.0, float("-inf")
    noise[6, 77] = 0.0                                                     # no number: nowhere the largest
    noise[7, x[7].argmax()] = float("inf")
    step = PagedStep.of([(1, 1, [0])] * 12, DEV)
    tree = PagedTree(step, torch.full((12,), -1, dtype=torch.int32, device=DEV))
    _, _, following = tree.accept(x.to(DEV), torch.zeros(12, dtype=torch.int32, device=DEV), temperature=temperature, noise=noise.to(DEV))
    want = T.targets(x, temperature, noise)
    assert following.tolist() == want and want[0] == 700 and want[2] == 5
