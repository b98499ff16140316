"""GPU: trees of drafted tokens over paged caches: what tokens see, attention, acceptance, rows that are kept, against plain 64-bit forms."""
import random

import pytest
import torch

import paged_oracle as O
import tree_oracle as T

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def setup(sequences, page, kv_heads, heads, dim, vdim, store, dtype, spare=2, seed=0):
    """(cache with everything written, q, step, [(new, length, pages)])."""
    from lit_llama_b200 import PagedCache, PagedStep

    g = torch.Generator().manual_seed(seed + 17)
    n_pages = sum(-(-length // page) for _, length in sequences) + spare
    seqs = O.random_pages(sequences, page, n_pages, g)
    cache = PagedCache.empty(n_pages, page, kv_heads, dim, vdim, dtype=dtype, store=store, device=DEV)
    total = sum(length for _, length in sequences)
    k, v = torch.randn(total, kv_heads, dim, generator=g).to(dtype).to(DEV), (torch.randn(total, kv_heads, vdim, generator=g) + 0.25).to(dtype).to(DEV)
    cache.write(k, v, PagedStep.of([(length, length, pages) for _, length, pages in seqs], DEV))
    step = PagedStep.of(seqs, DEV)
    q = torch.randn(step.rows, heads, dim, generator=g).to(dtype).to(DEV)
    return cache, q, step, seqs


def trees_of(seqs, rng):
    return [T.random_parents(n, rng) for n, _, _ in seqs]


def flat(trees):
    return torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=DEV)


def sights(seqs, trees, window=0, first=0):
    sets, depths = [], []
    for (n, length, _), parents in zip(seqs, trees):
        for s, d in T.ancestors(parents, window, first, length - n):
            sets.append(s)
            depths.append(d)
    return sets, depths


def check(got, want, size, keys, f32, store):
    out, mag, dots = want
    bound = O.tolerance(out, mag, dots, size, keys, f32, store)
    err = (got.cpu().to(O.F64) - out).abs()
    assert bool((err <= bound).all()), float((err / bound).max())


# ----------------------------------------------------------------------------- what tokens see
@pytest.mark.parametrize("window,first", [(0, 0), (3, 0), (2, 21), (1, 0)])
def test_masks_depths_and_positions(window, first):
    from lit_llama_b200 import PagedStep, PagedTree

    rng = random.Random(5)
    seqs = [(n, n + c, [0] * 40) for n, c in ((7, 13), (0, 9), (1, 0), (70, 20), (33, 2))]
    trees = trees_of(seqs, rng)
    trees[0][3], trees[0][4], trees[3][9], trees[3][40] = 3, 6, -5, 2 ** 31 - 1      # not before the token: none
    step = PagedStep.of(seqs, DEV)
    tree = PagedTree(step, flat(trees), window=window, first=first)
    sets, depths = sights(seqs, trees, window, first)
    assert tree.words == 3 and torch.equal(tree.masks.cpu(), T.bits(sets, 3)) and tree.depths.tolist() == depths
    base = [length - n for n, length, _ in seqs for _ in range(n)]
    assert tree.positions.tolist() == [b + d for b, d in zip(base, depths)]
    # contents overwritten, rows of no sequence
    step.starts.copy_(torch.tensor([2, 7, 7, 8, 78, 100]))
    tree.update()
    sets, depths = sights([(5, 20, []), (0, 9, []), (1, 1, []), (70, 90, []), (22, 35, [])], [tree.parents.tolist()[a:b] for a, b in ((2, 7), (7, 7), (7, 8), (8, 78), (78, 100))], window, first)
    empty = [set()] * 2, [0] * 2
    assert torch.equal(tree.masks.cpu(), T.bits(empty[0] + sets + [set()] * 11, 3)) and tree.depths.tolist() == [0, 0] + depths + [0] * 11


# ----------------------------------------------------------------------------- attention
CASES = [
    # sequences (new, length); page, kv_heads, heads, dim, vdim
    ([(1, 1)], 16, 1, 1, 64, 64),
    ([(5, 5)], 16, 2, 8, 128, 128),
    ([(8, 203)], 64, 4, 4, 128, 128),
    ([(13, 130), (1, 77), (0, 5), (16, 16), (3, 300)], 16, 2, 4, 64, 32),
    ([(64, 700)], 32, 1, 4, 128, 128),
    ([(33, 333), (40, 41), (2, 500)], 128, 2, 16, 128, 64),
    ([(100, 612), (97, 140)], 64, 1, 8, 192, 128),
    ([(300, 301), (7, 900)], 256, 1, 2, 80, 48),
    ([(9, 150), (20, 90)], 16, 2, 6, 256, 256),
]


@pytest.mark.parametrize("store,dtype", [("act", BF), ("fp8", BF), ("int8", BF), ("act", F32), ("fp8", F32), ("int8", F32)], ids=str)
@pytest.mark.parametrize("case", range(len(CASES)))
def test_attention_over_context_and_ancestors(case, store, dtype):
    from lit_llama_b200 import PagedTree

    sequences, page, kv, heads, dim, vdim = CASES[case]
    cache, q, step, seqs = setup(sequences, page, kv, heads, dim, vdim, store, dtype, seed=case)
    trees = trees_of(seqs, random.Random(case))
    tree = PagedTree(step, flat(trees))
    sets, depths = sights(seqs, trees)
    want = T.attend(q, cache, seqs, sets, depths, dim ** -0.5)
    check(cache.attend(q, step, tree=tree), want, dim, max(m for _, m in sequences), dtype == F32, store)


def steered(seqs, group, form):
    """The same step with hints that make the call take one of its forms: few rows at a time, row tiles of 128 rows, of 256.  (A wide table: many keys, as far as the host knows.)"""
    from lit_llama_b200 import PagedStep

    step = PagedStep.of(seqs, DEV, width=8192)
    new = {"few": max(16 // group, 1), "pair": max(128 // group, 1), "many": 4096}[form]
    return PagedStep(step.starts, step.lengths, step.table, rows=step.rows, max_new=new)


@pytest.mark.parametrize("store", ["act", "fp8", "int8"])
@pytest.mark.parametrize("form", ["few", "pair", "many"])
@pytest.mark.parametrize("case", range(len(CASES) - 1))
def test_every_form_is_right(case, form, store):
    """Whatever the hints say: trees of more rows than a form is chosen for, and of fewer."""
    from lit_llama_b200 import PagedTree

    sequences, page, kv, heads, dim, vdim = CASES[case]
    cache, q, _, seqs = setup(sequences, page, kv, heads, dim, vdim, store, BF, seed=case)
    step = steered(seqs, heads // kv, form)
    trees = trees_of(seqs, random.Random(case))
    tree = PagedTree(step, flat(trees), nodes=max(n for n, _ in sequences))
    sets, depths = sights(seqs, trees)
    check(cache.attend(q, step, tree=tree), T.attend(q, cache, seqs, sets, depths, dim ** -0.5), dim, max(m for _, m in sequences), False, store)


@pytest.mark.parametrize("store", ["act", "fp8", "int8"])
@pytest.mark.parametrize("form", ["pair", "many"])
@pytest.mark.parametrize("dim,vdim,page", [(16, 16, 16), (192, 128, 64), (176, 112, 32), (48, 128, 128), (96, 16, 256), (32, 80, 16)])
def test_sizes_of_heads_in_row_tiles(dim, vdim, page, form, store):
    from lit_llama_b200 import PagedTree

    sequences = [(20, 700), (9, 128), (32, 290), (1, 129), (3, 3)]
    cache, q, _, seqs = setup(sequences, page, 2, 8, dim, vdim, store, BF, seed=dim)
    step = steered(seqs, 4, form)
    trees = trees_of(seqs, random.Random(dim))
    tree = PagedTree(step, flat(trees), nodes=32)
    sets, depths = sights(seqs, trees)
    check(cache.attend(q, step, tree=tree), T.attend(q, cache, seqs, sets, depths, dim ** -0.5), dim, 700, False, store)


@pytest.mark.parametrize("store", ["act", "fp8"])
@pytest.mark.parametrize("form", ["pair", "many"])
@pytest.mark.parametrize("keys", [1, 100, 128, 129, 256, 257, 384, 640])
def test_one_tile_of_keys_two_and_more(keys, form, store):
    """Row tiles whose halves have none, one or several tiles of keys."""
    from lit_llama_b200 import PagedTree

    sequences = [(min(keys, 12), keys), (min(keys, 30), keys), (1, keys)]
    cache, q, _, seqs = setup(sequences, 64, 1, 4, 64, 64, store, BF, seed=keys)
    step = steered(seqs, 4, form)
    trees = trees_of(seqs, random.Random(keys))
    tree = PagedTree(step, flat(trees), nodes=30)
    sets, depths = sights(seqs, trees)
    check(cache.attend(q, step, tree=tree), T.attend(q, cache, seqs, sets, depths, 64 ** -0.5), 64, keys, False, store)


@pytest.mark.parametrize("store", ["act", "int8"])
@pytest.mark.parametrize("form", ["pair", "many"])
@pytest.mark.parametrize("window,first", [(1, 0), (40, 0), (64, 5), (130, 300), (300, 16)])
def test_windows_in_row_tiles(window, first, form, store):
    from lit_llama_b200 import PagedTree

    sequences = [(21, 900), (6, 40), (1, 600), (12, 12), (30, 1000)]
    cache, q, _, seqs = setup(sequences, 16, 1, 4, 64, 64, store, BF)
    step = steered(seqs, 4, form)
    trees = trees_of(seqs, random.Random(window))
    tree = PagedTree(step, flat(trees), nodes=30, window=window, first=first)
    sets, depths = sights(seqs, trees, window, first)
    check(cache.attend(q, step, tree=tree, window=window, first=first), T.attend(q, cache, seqs, sets, depths, 64 ** -0.5, window, first), 64, 1000, False, store)


@pytest.mark.parametrize("store", ["act", "fp8", "int8"])
@pytest.mark.parametrize("form", ["pair", "many"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_bad_rows_and_odd_masks_in_row_tiles(bad, form, store):
    """Tokens that see nothing or later ones, depths out of range, pages that are not there, and a value that is no number: only rows that see it have it."""
    from lit_llama_b200 import PagedStep, PagedTree

    sequences = [(25, 25), (28, 400), (5, 80)]
    cache, q, _, seqs = setup(sequences, 16, 2, 8, 64, 64, store, BF)
    k, v = cache.read(PagedStep.of([(400, 400, seqs[1][2])], DEV))
    k[380], v[380] = bad, bad                                              # new token 8 of the second
    cache.write(k, v, PagedStep.of([(400, 400, seqs[1][2])], DEV))
    seqs[1] = (28, 400, [-1 if i in (2, 3, 4, 5, 6, 7, 8, 9, 20) else p for i, p in enumerate(seqs[1][2])])
    step = steered(seqs, 4, form)
    tree = PagedTree(step, flat(trees_of(seqs, random.Random(1))), nodes=28)
    rng = random.Random(2)
    sets = [{i for i in range(32) if rng.random() < 0.3} for _ in range(step.rows)]
    for r in (0, 3, 24):
        sets[r] = set()
    hit = [r for r in range(25, 53) if 8 in sets[r]]
    spared = [r for r in range(58) if r not in hit]
    tree.masks.copy_(T.bits(sets, 1))
    depths = [rng.choice([-3, 0, 1, 4, 1000]) for _ in range(step.rows)]
    tree.depths.copy_(torch.tensor(depths, dtype=torch.int32))
    got = cache.attend(q, step, tree=tree, window=300, first=40)
    assert hit and not torch.isfinite(got[hit]).any() and not got[[0, 3, 24]].any()
    want = T.attend(q, cache, seqs, [s - {8} if 25 <= r < 53 else s for r, s in enumerate(sets)], depths, 64 ** -0.5, 300, 40)
    check(got[spared], tuple(x[spared] for x in want), 64, 400, False, store)


@pytest.mark.parametrize("store,dtype", [("act", BF), ("int8", BF), ("act", F32)], ids=str)
@pytest.mark.parametrize("window,first", [(1, 0), (40, 0), (64, 5), (33, 70), (500, 16)])
@pytest.mark.parametrize("group", [1, 4, 16])
def test_windows_count_from_the_position_in_the_tree(group, window, first, store, dtype):
    from lit_llama_b200 import PagedTree

    sequences = [(21, 333), (6, 40), (1, 200), (12, 12)]
    cache, q, step, seqs = setup(sequences, 16, 1, group, 64, 64, store, dtype)
    trees = trees_of(seqs, random.Random(group))
    tree = PagedTree(step, flat(trees), window=window, first=first)
    sets, depths = sights(seqs, trees, window, first)
    want = T.attend(q, cache, seqs, sets, depths, 64 ** -0.5, window, first)
    check(cache.attend(q, step, tree=tree, window=window, first=first), want, 64, 333, dtype == F32, store)


@pytest.mark.parametrize("store,dtype", [("act", BF), ("fp8", BF), ("int8", BF), ("act", F32)], ids=str)
@pytest.mark.parametrize("sequences,window", [([(8, 300)], 0), ([(70, 200), (3, 4), (1, 600)], 0), ([(40, 400), (5, 77)], 100)])
def test_a_chain_is_what_causal_attention_gives(sequences, window, store, dtype):
    """Against the causal formula itself.  (Not bit by bit against the causal call: a row tile of a tree goes on to the sequence's last key, one of causal rows to its
    last row's, so the keys are shared among warps otherwise and f32 sums are added in another order: each within the bound.)"""
    from lit_llama_b200 import PagedTree

    cache, q, step, seqs = setup(sequences, 32, 2, 8, 128, 64, store, dtype)
    tree = PagedTree(step, flat([[i - 1 for i in range(n)] for n, _, _ in seqs]), window=window)
    want = O.attend(q, cache, seqs, 128 ** -0.5, window)
    for got in (cache.attend(q, step, tree=tree, window=window), cache.attend(q, step, window=window)):
        check(got, want, 128, 600, dtype == F32, store)


@pytest.mark.parametrize("store,dtype", [("act", BF), ("fp8", BF), ("act", F32)], ids=str)
@pytest.mark.parametrize("heads", [2, 8])
def test_any_masks_and_depths(heads, store, dtype):
    """Masks written over: tokens that see nothing at all, later ones, bits behind the last token; depths out of range."""
    from lit_llama_b200 import PagedTree

    sequences = [(37, 37), (5, 80), (64, 64)]
    cache, q, step, seqs = setup(sequences, 16, 2, heads, 64, 64, store, dtype)
    tree = PagedTree(step, flat(trees_of(seqs, random.Random(1))))
    rng = random.Random(2)
    sets = [{i for i in range(64) if rng.random() < 0.3} for _ in range(step.rows)]
    for r in (0, 3, 36, 50, 99):
        sets[r] = set()
    depths = [rng.choice([-3, 0, 1, 4, 1000]) for _ in range(step.rows)]
    tree.masks.copy_(T.bits(sets, 2))
    tree.depths.copy_(torch.tensor(depths, dtype=torch.int32))
    for window, first in ((0, 0), (30, 3)):
        got = cache.attend(q, step, tree=tree, window=window, first=first)
        check(got, T.attend(q, cache, seqs, sets, depths, 64 ** -0.5, window, first), 64, 80, dtype == F32, store)
        assert not got[[0, 3, 36, 50, 99]].any()


@pytest.mark.parametrize("store,dtype", [("act", BF), ("fp8", BF), ("int8", BF), ("act", F32)], ids=str)
@pytest.mark.parametrize("heads", [2, 8])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_a_token_does_not_see_does_not_reach_it(bad, heads, store, dtype):
    """A drafted token's key and value that are NaN or infinite: its descendants have them, its siblings do not."""
    from lit_llama_b200 import PagedStep, PagedTree

    sequences = [(20, 60)]
    cache, q, step, seqs = setup(sequences, 16, 2, heads, 64, 64, store, dtype)
    parents = [-1, 0, 0] + [1 if i % 2 else 2 for i in range(3, 20)]
    tree = PagedTree(step, flat([parents]))
    sets, depths = sights(seqs, [parents])
    hit = [i for i in range(20) if 1 in sets[i]]
    spared = [i for i in range(20) if 1 not in sets[i]]
    k, v = cache.read(PagedStep.of([(60, 60, seqs[0][2])], DEV))
    clean = T.attend(q, cache, seqs, sets, depths, 64 ** -0.5)
    k[41], v[41] = bad, bad
    cache.write(k, v, PagedStep.of([(60, 60, seqs[0][2])], DEV))
    got = cache.attend(q, step, tree=tree)
    assert not torch.isfinite(got[hit]).any()
    # rows written back are quantised again: an 8-bit row is off by another half step
    if store == "act":
        check(got[spared], tuple(x[spared] for x in clean), 64, 60, dtype == F32, store)
    else:
        again = [x for x in T.attend(q, cache, seqs, [s - {1} for s in sets], depths, 64 ** -0.5)]
        check(got[spared], tuple(x[spared] for x in again), 64, 60, dtype == F32, store)


@pytest.mark.parametrize("store,dtype", [("act", BF), ("int8", BF), ("act", F32)], ids=str)
@pytest.mark.parametrize("parts,dim,vdim", [(2, 64, 80), (3, 64, 80), (4, 256, 256), (5, 64, 80), (6, 64, 80), (7, 64, 80), (8, 64, 80), (8, 256, 192), (9, 64, 80), (12, 64, 80)])
def test_keys_in_any_number_of_parts(parts, dim, vdim, store, dtype):
    """Two sequences that have so many parts of 128 keys, and a last part of another size; then a token that some rows see and others do not is NaN."""
    from lit_llama_b200 import PagedStep, PagedTree

    sequences = [(5, 128 * parts + 40), (3, 60)]
    cache, q, step, seqs = setup(sequences, 16, 2, 4, dim, vdim, store, dtype)
    parents = [-1, 0, 0, 1, 2, -1, 0, 1]
    tree = PagedTree(step, torch.tensor(parents, dtype=torch.int32, device=DEV))
    sets, depths = sights(seqs, [parents[:5], parents[5:]])
    want = T.attend(q, cache, seqs, sets, depths, dim ** -0.5)
    check(cache.attend(q, step, tree=tree), want, dim, 128 * parts + 40, dtype == F32, store)
    again = PagedStep.of([(length, length, pages) for _, length, pages in seqs], DEV)
    k, v = cache.read(again)
    k[sequences[0][1] - 4], v[sequences[0][1] - 4] = float("nan"), float("inf")      # the first tree's token 1
    cache.write(k, v, again)
    got = cache.attend(q, step, tree=tree)
    hit = [1, 3]
    spared = [r for r in range(8) if r not in hit]
    assert not torch.isfinite(got[hit]).any()
    hidden = T.attend(q, cache, seqs, [s - {1} if r < 5 else s for r, s in enumerate(sets)], depths, dim ** -0.5)
    check(got[spared], tuple(x[spared] for x in hidden), dim, 128 * parts + 40, dtype == F32, store)


@pytest.mark.parametrize("store", ["act", "fp8"])
@pytest.mark.parametrize("new", [3, 40])
def test_pages_that_are_not_there_and_rows_behind_the_last_sequence(new, store):
    from lit_llama_b200 import PagedStep, PagedTree

    cache, q, step, seqs = setup([(new, 150), (1, 30)], 16, 2, 8, 64, 64, store, BF)
    gone = [(n, length, [-1 if i in (0, 4) else p for i, p in enumerate(pages)]) for n, length, pages in seqs]
    gone[1] = (1, 30, [cache.n_pages, -7])
    step = PagedStep.of(gone, DEV)
    trees = trees_of(gone, random.Random(3))
    tree = PagedTree(step, flat(trees))
    sets, depths = sights(gone, trees)
    want = T.attend(q, cache, gone, sets, depths, 64 ** -0.5)
    more = torch.cat([q, q[:2]])
    got = cache.attend(more, step, tree=tree)
    assert got.shape[0] == new + 3 and not got[new:].any()
    check(got[:new + 1], want, 64, 150, False, store)
    out = torch.full_like(got, 7.0)
    assert cache.attend(more, step, tree=tree, out=out) is out
    assert torch.equal(out[:new + 1], got[:new + 1]) and bool((out[new + 1:] == 7.0).all())
    # the step's tensors overwritten: the first rows and the last belong to no sequence
    step.starts.copy_(torch.tensor([1, new, new], dtype=torch.int32))
    tree.update()
    got = cache.attend(more, step, tree=tree)
    assert not got[0].any() and not got[new:].any()
    out.fill_(7.0)
    cache.attend(more, step, tree=tree, out=out)
    assert bool((out[0] == 7.0).all()) and bool((out[new:] == 7.0).all()) and torch.equal(out[1:new], got[1:new])


@pytest.mark.parametrize("store", ["fp8", "int8"])
@pytest.mark.parametrize("new", [6, 70])
def test_a_tree_among_many_single_tokens(new, store):
    """Enough of them that the step runs the kernels of few and of many rows side by side (from 8-bit pools)."""
    from lit_llama_b200 import PagedTree

    sequences = [(1, 2000 + 10 * b) for b in range(60)]
    sequences[7] = (new, 1200)
    cache, q, step, seqs = setup(sequences, 64, 8, 32, 32, 32, store, BF)
    trees = trees_of(seqs, random.Random(6))
    tree = PagedTree(step, flat(trees))
    got = cache.attend(q, step, tree=tree)
    some = [0, 7, 30, 59]                                                   # of the oracle's, some sequences
    at = [sum(n for n, _ in sequences[:b]) for b in range(61)]
    rows = [r for b in some for r in range(at[b], at[b + 1])]
    sets, depths = sights([seqs[b] for b in some], [trees[b] for b in some])
    want = T.attend(q[rows], cache, [seqs[b] for b in some], sets, depths, 32 ** -0.5)
    check(got[rows], want, 32, 3000, False, store)


def test_rows_of_logits_far_apart():
    """Rows whose distance passes 32 bits."""
    from lit_llama_b200 import PagedStep, PagedTree, beam_select

    far = 3 * 2 ** 29
    big = torch.empty(2 * far + 5000, dtype=BF, device=DEV)
    x = big.as_strided((3, 5000), (far, 1))
    x.copy_(torch.randn(3, 5000, device=DEV))
    tree = PagedTree(PagedStep.of([(1, 1, [0])] * 3, DEV), torch.full((3,), -1, dtype=torch.int32, device=DEV))
    assert tree.accept(x, torch.zeros(3, dtype=torch.int64, device=DEV))[2].tolist() == T.targets(x)
    scores = torch.zeros(1, 3, device=DEV)
    got, want = beam_select(x[None], scores, 12), beam_select(x.contiguous()[None], scores, 12)
    assert all(torch.equal(a, b) for a, b in zip(got[1:], want[1:]))


@pytest.mark.parametrize("heads", [2, 8])
def test_queries_as_large_as_f32_goes(heads):
    """Rounded to bf16 the largest f32 are infinities: the parts a query is computed in are not.  The keys have few bits and are as small as their products ask for."""
    from lit_llama_b200 import PagedStep, PagedTree

    cache, q, step, seqs = setup([(9, 150)], 16, 2, heads, 16, 32, "act", F32)
    g = torch.Generator().manual_seed(3)
    k = (torch.randint(2, 8, (150, 2, 16), generator=g) * (torch.randint(0, 2, (150, 2, 16), generator=g) * 2 - 1)).to(F32) * 2.0 ** -128
    cache.write(k.to(DEV), torch.randn(150, 2, 32, generator=g).to(DEV), PagedStep.of([(150, 150, seqs[0][2])], DEV))
    most = torch.finfo(F32).max
    q = ((torch.rand(9, heads, 16, generator=g) * 0.01 + 0.99).clamp(max=1.0) * most * (torch.randint(0, 2, (9, heads, 16), generator=g) * 2 - 1)).to(DEV)
    q[::2, :, 3] = most
    trees = trees_of(seqs, random.Random(heads))
    sets, depths = sights(seqs, trees)
    want = T.attend(q, cache, seqs, sets, depths, 16 ** -0.5)
    check(cache.attend(q, step, tree=PagedTree(step, flat(trees))), want, 16, 150, True, "act")


def test_queries_of_any_stride():
    from lit_llama_b200 import PagedTree

    cache, q, step, seqs = setup([(24, 100)], 16, 2, 8, 64, 64, "act", BF)
    tree = PagedTree(step, flat(trees_of(seqs, random.Random(4))))
    want = cache.attend(q, step, tree=tree)
    wide = torch.zeros(24, 8 * 64 + 40, dtype=BF, device=DEV)
    wide[:, 8:8 + 512] = q.view(24, 512)
    for x in (wide[:, 8:520].unflatten(1, (8, 64)), q.transpose(0, 1).contiguous().transpose(0, 1), wide.new_empty(24 * 512 + 1)[1:].view(24, 8, 64).copy_(q)):
        assert torch.equal(cache.attend(x, step, tree=tree), want)


# ----------------------------------------------------------------------------- acceptance
def planted(trees, vocab, dtype, rng, agree=0.7):
    """Logits and tokens where most tokens are what their parent's row has as its largest."""
    rows = sum(len(t) for t in trees)
    x = torch.randn(rows, vocab) * 2
    tokens = [rng.randrange(vocab) for _ in range(rows)]
    at = 0
    for t in trees:
        for p in range(len(t)):
            children = [j for j in range(p + 1, len(t)) if t[j] == p]
            if children and rng.random() < agree:
                x[at + p, tokens[at + rng.choice(children)]] = 20.0
        at += len(t)
    return x.to(dtype).to(DEV), tokens


@pytest.mark.parametrize("vocab,dtype,wide", [(1, F32, True), (7, BF, False), (255, F32, False), (4096, BF, True), (4097, BF, False), (32000, F32, True), (100003, BF, True)], ids=str)
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_accepted_paths(temperature, vocab, dtype, wide):
    from lit_llama_b200 import PagedStep, PagedTree

    rng = random.Random(vocab)
    seqs = [(n, n + 3, [0] * 8) for n in (8, 1, 0, 40, 77, 2)]
    trees = trees_of(seqs, rng)
    step = PagedStep.of(seqs, DEV)
    logits, tokens = planted(trees, vocab, dtype, rng)
    noise = torch.empty(step.rows, vocab, device=DEV).exponential_(1) if temperature else None
    tree = PagedTree(step, flat(trees))
    kept, counts, following = tree.accept(logits, torch.tensor(tokens, dtype=torch.int64 if wide else torch.int32, device=DEV), temperature=temperature, noise=noise)
    target = T.targets(logits, temperature, noise)
    at, want, n, nxt = 0, [], [], []
    for t in trees:
        path, last = T.accept(target[at:at + len(t)], tokens[at:at + len(t)], t)
        want += path + [-1] * (len(t) - len(path))
        n.append(len(path))
        nxt.append(last)
        at += len(t)
    assert kept.tolist() == want and counts.tolist() == n and following.tolist() == nxt
    assert vocab < 100 or max(n) > 1                                       # some drafts are taken


def test_acceptance_of_logits_that_are_no_numbers_and_of_ties():
    from lit_llama_b200 import PagedStep, PagedTree

    step = PagedStep.of([(1, 1, [0])] * 7, DEV)
    tree = PagedTree(step, torch.full((7,), -1, dtype=torch.int32, device=DEV))
    x = torch.randn(7, 5001, device=DEV)
    nan, inf = float("nan"), float("inf")
    x[0] = -inf
    x[1] = nan
    x[2, 17], x[2, 4100] = nan, 50.0
    x[3, 4999], x[3, 30] = inf, inf
    x[4] = 3.0
    x[5] = -inf
    x[5, 5000] = -1e30
    x[6, 11], x[6, 10] = 0.0, -0.0
    x[6, :10] = -1.0
    x[6, 12:] = -1.0
    tokens = torch.zeros(7, dtype=torch.int64, device=DEV)
    want = [0, 0, 4100, 30, 0, 5000, 10]
    for y in (x, x.to(BF)):
        assert tree.accept(y, tokens)[2].tolist() == want
        ones = torch.ones(7, 5001, device=DEV)
        assert tree.accept(y, tokens, temperature=0.5, noise=ones)[2].tolist() == want
    noise = torch.ones(7, 5001, device=DEV)
    noise[:, 321] = 0.0                                                    # the smallest there can be: always chosen, where its logit is above -inf
    assert tree.accept(x, tokens, temperature=1.0, noise=noise)[2].tolist() == [0, 0, 321, 30, 321, 5000, 321]


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("mask", [float("-inf"), None])
@pytest.mark.parametrize("temperature", [1.0, 0.5, 1e-39])
def test_acceptance_of_a_vocabulary_that_is_hidden_but_for_a_few(temperature, mask, dtype):
    from lit_llama_b200 import PagedStep, PagedTree

    rows, vocab = 9, 20011
    tree = PagedTree(PagedStep.of([(1, 1, [0])] * rows, DEV), torch.full((rows,), -1, dtype=torch.int32, device=DEV))
    g = torch.Generator().manual_seed(8)
    mask = torch.finfo(dtype).min if mask is None else mask
    x = torch.full((rows, vocab), mask, dtype=dtype)
    noise = torch.empty(rows, vocab).exponential_(1, generator=g)
    for r in range(5):                                                     # some few left, the next four rows have none or a curious one
        at = torch.randint(0, vocab, (r + 1,), generator=g)
        x[r, at] = torch.randn(r + 1, generator=g).to(dtype)
    noise[6, :9000], noise[7, 12345] = float("inf"), 0.0
    x[8] = torch.where(torch.arange(vocab) % 3 == 0, -0.0, x[8].float()).to(dtype)
    x[8, 3000:] = mask
    tokens = torch.zeros(rows, dtype=torch.int64, device=DEV)
    assert tree.accept(x.to(DEV), tokens, temperature=temperature, noise=noise.to(DEV))[2].tolist() == T.targets(x, temperature, noise)


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_logits_and_noise_of_any_stride(dtype):
    from lit_llama_b200 import PagedStep, PagedTree

    rng = random.Random(9)
    seqs = [(12, 12, [0]), (3, 9, [0])]
    trees = trees_of(seqs, rng)
    step = PagedStep.of(seqs, DEV)
    tree = PagedTree(step, flat(trees))
    x, tokens = planted(trees, 999, dtype, rng)
    tokens = torch.tensor(tokens, device=DEV)
    noise = torch.empty(15, 999, device=DEV).exponential_(1)
    for temperature, nz in ((0.0, None), (0.9, noise)):
        want = [t.tolist() for t in tree.accept(x, tokens, temperature=temperature, noise=nz)]
        big = torch.full((17, 1024), 99.0, dtype=dtype, device=DEV)
        big[:15, 3:1002] = x
        nz2 = None
        if nz is not None:
            nz2 = torch.zeros(15, 1001, device=DEV)
            nz2[:, 1:1000] = nz
            nz2 = nz2[:, 1:1000]
        for y in (big[:, 3:1002], x.t().contiguous().t(), torch.cat([x, x])):
            assert [t.tolist() for t in tree.accept(y, tokens, temperature=temperature, noise=nz2)] == want
    counts = torch.zeros(5, dtype=torch.int64)
    for _ in range(200):                                                   # drawn without noise given: as often as the softmax says
        one = PagedTree(PagedStep.of([(40, 40, [0, 0, 0])], DEV), torch.full((40,), -1, dtype=torch.int32, device=DEV))
        counts[int(one.accept(torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5]], device=DEV).expand(40, 5), torch.zeros(40, dtype=torch.int64, device=DEV), temperature=1.0)[2])] += 1
    p = torch.softmax(torch.tensor([0.0, 1.0, 2.0, -1.0, 0.5]), 0)
    assert bool(((counts / 200 - p).abs() < 6 * (p * (1 - p) / 200).sqrt()).all())      # six standard deviations


# ----------------------------------------------------------------------------- rows that are kept
def raw(t):
    return t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t


@pytest.mark.parametrize("store,dtype", [("act", BF), ("fp8", BF), ("int8", BF), ("act", F32), ("int8", F32)], ids=str)
@pytest.mark.parametrize("layers,page,kv,dim,vdim", [(1, 16, 1, 16, 16), (3, 32, 2, 128, 64), (70, 16, 3, 48, 32), (2, 128, 40, 64, 256)])
def test_kept_rows_move_together(layers, page, kv, dim, vdim, store, dtype):
    from lit_llama_b200 import PagedCache, PagedLayers, PagedStep

    rng = random.Random(layers)
    sequences = [(30, 100), (0, 20), (1, 17), (90, 130), (12, 12), (5, 40)]
    n_pages = sum(-(-m // page) for _, m in sequences) + 1
    seqs = O.random_pages(sequences, page, n_pages, torch.Generator().manual_seed(3))
    seqs[5] = (5, 40, [-1] + seqs[5][2][1:]) if page == 16 else seqs[5]
    caches = []
    for _ in range(layers):
        c = PagedCache.empty(n_pages, page, kv, dim, vdim, dtype=dtype, store=store, device=DEV)
        for t in c._pool:
            if t is not None:
                raw(t).copy_(torch.randint(-100, 100, t.shape, device=DEV).to(raw(t).dtype))
        caches.append(c)
    before = [[raw(t).clone() if t is not None else None for t in c._pool] for c in caches]
    paths = [sorted(rng.sample(range(n), rng.randint(1, n))) if n else [] for n, _, _ in seqs]
    paths[3] = [0] + sorted(rng.sample(range(1, 90), 70))                  # more than are looked up at a time
    kept = torch.tensor([k for (n, _, _), p in zip(seqs, paths) for k in p + [-1] * (n - len(p))], dtype=torch.int32, device=DEV)
    counts = torch.tensor([len(p) for p in paths], dtype=torch.int32, device=DEV)
    PagedLayers(caches).keep(PagedStep.of(seqs, DEV), kept, counts)
    for c, was in zip(caches, before):
        for t, w in zip(c._pool, was):
            if t is None:
                continue
            want = w.clone()
            for (n, length, pages), path in zip(seqs, paths):
                for i, k in enumerate(path):
                    (pf, f), (pt, to) = divmod(length - n + k, page), divmod(length - n + i, page)
                    if pages[pf] >= 0 and pages[pt] >= 0:
                        want[pages[pt], :, to] = w[pages[pf], :, f]
            assert torch.equal(raw(t), want)


def test_kept_places_outside_the_new_tokens_are_left_out():
    from lit_llama_b200 import PagedCache, PagedLayers, PagedStep

    c = PagedCache.empty(2, 16, 1, 16, device=DEV)
    c.k.normal_()
    k = c.k.clone()
    step = PagedStep.of([(4, 20, [1, 0])], DEV)
    PagedLayers([c]).keep(step, torch.tensor([7, -1, 3, 2 ** 31 - 1], dtype=torch.int32, device=DEV), torch.tensor([9], dtype=torch.int32, device=DEV))
    k[0, :, 2] = k[0, :, 3]
    assert torch.equal(c.k, k)


@pytest.mark.parametrize("store,dtype", [("act", BF), ("fp8", BF), ("int8", F32)], ids=str)
@pytest.mark.parametrize("layers,page,kv,dim,vdim", [(1, 16, 1, 16, 16), (66, 16, 3, 48, 32), (2, 256, 40, 64, 256), (3, 64, 8, 128, 128)])
def test_pages_are_copied_in_all_layers(layers, page, kv, dim, vdim, store, dtype):
    from lit_llama_b200 import PagedCache, PagedLayers

    caches = []
    for _ in range(layers):
        c = PagedCache.empty(9, page, kv, dim, vdim, dtype=dtype, store=store, device=DEV)
        for t in c._pool:
            if t is not None:
                raw(t).copy_(torch.randint(-100, 100, t.shape, device=DEV).to(raw(t).dtype))
        caches.append(c)
    before = [[raw(t).clone() if t is not None else None for t in c._pool] for c in caches]
    pairs = [(0, 5), (0, 8), (3, 1), (7, 2)]
    layers_ = PagedLayers(caches)
    layers_.copy(pairs)
    layers_.copy(torch.tensor([[2, 2], [-1, 3], [4, 9], [9, 4], [2 ** 31 - 1, 0]], dtype=torch.int32, device=DEV))      # left out
    layers_.copy([])
    for c, was in zip(caches, before):
        for t, w in zip(c._pool, was):
            if t is not None:
                for a, b in pairs:
                    w[b] = w[a]
                assert torch.equal(raw(t), w)


# ----------------------------------------------------------------------------- together, in graphs, on other streams
def test_a_step_with_drafts_recorded_and_replayed_with_other_contents():
    """Rotation apart, what a step with drafts does: what tokens see, rows written, attention, acceptance, rows kept, in one graph; then other trees, lengths and logits."""
    from lit_llama_b200 import PagedCache, PagedLayers, PagedStep, PagedTree

    def world(seed):
        rng = random.Random(seed)
        sequences = [(9, 40 + seed), (9, 100), (9, 9 + 3 * seed)]
        seqs = O.random_pages(sequences, 16, 24, torch.Generator().manual_seed(seed))
        trees = trees_of(seqs, rng)
        torch.manual_seed(seed)                                            # the same world whenever it is made
        logits, tokens = planted(trees, 500, BF, rng)
        g = torch.Generator().manual_seed(seed)
        return seqs, trees, logits, tokens, [torch.randn(27, n, 64, generator=g).to(BF).to(DEV) for n in (2, 2, 8)]

    def fresh():
        caches = [PagedCache.empty(24, 16, 2, 64, dtype=BF, store="int8", device=DEV) for _ in range(2)]
        for i, c in enumerate(caches):
            g = torch.Generator().manual_seed(40 + i)
            c.write(torch.randn(384, 2, 64, generator=g).to(BF).to(DEV), torch.randn(384, 2, 64, generator=g).to(BF).to(DEV), PagedStep.of([(384, 384, list(range(24)))], DEV))
        return caches, PagedLayers(caches)

    def body(caches, layers, step, tree, k, v, q, logits, tokens):
        tree.update()
        outs = []
        for c in caches:
            c.write(k, v, step)
            outs.append(c.attend(q, step, tree=tree))
        kept, counts, following = tree.accept(logits, tokens)
        layers.keep(step, kept, counts)
        return outs + [kept, counts, following]

    def eager(seed):
        seqs, trees, logits, tokens, (k, v, q) = world(seed)
        caches, layers = fresh()
        step = PagedStep.of(seqs, DEV, width=12)
        out = body(caches, layers, step, PagedTree(step, flat(trees)), k, v, q, logits, torch.tensor(tokens, device=DEV))
        return out + [t for c in caches for t in c._pool]

    seqs, trees, logits, tokens, (k, v, q) = world(1)
    caches, layers = fresh()
    step = PagedStep.of(seqs, DEV, width=12)
    tree, tokens = PagedTree(step, flat(trees)), torch.tensor(tokens, device=DEV)
    body(caches, layers, step, tree, k, v, q, logits, tokens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = body(caches, layers, step, tree, k, v, q, logits, tokens)
    for seed in (2, 7, 1):
        seqs, trees, logits2, tokens2, qkv = world(seed)
        again, _ = fresh()
        for c, d in zip(caches, again):
            for t, u in zip(c._pool, d._pool):
                t.copy_(u)
        step.refill(PagedStep.of(seqs, DEV))
        tree.parents.copy_(flat(trees))
        for a, b in zip((logits, tokens, k, v, q), (logits2, torch.tensor(tokens2, device=DEV), *qkv)):
            a.copy_(b)
        graph.replay()
        want = eager(seed)
        for a, b in zip(got + [t for c in caches for t in c._pool], want):
            assert torch.equal(raw(a), raw(b)), seed


def test_calls_on_two_streams_at_once():
    from lit_llama_b200 import PagedTree, beam_select

    made = [setup([(24, 900), (40, 300)], 16, 2, 8, 64, 64, "act", BF, seed=s) for s in (1, 2)]
    trees = [PagedTree(m[2], flat(trees_of(m[3], random.Random(i)))) for i, m in enumerate(made)]
    logits = [torch.randn(4, 8, 32000, device=DEV) for _ in range(2)]
    scores = [torch.randn(4, 8, device=DEV) for _ in range(2)]
    rows = [torch.randn(64, 32000, device=DEV) for _ in range(2)]
    tokens = torch.zeros(64, dtype=torch.int64, device=DEV)

    def call(i):
        cache, q, step, _ = made[i]
        return [cache.attend(q, step, tree=trees[i]), *beam_select(logits[i], scores[i], 16), *trees[i].accept(rows[i], tokens)]

    want = [call(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append(call(i))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_steps_without_rows_or_sequences():
    from lit_llama_b200 import PagedCache, PagedLayers, PagedStep, PagedTree

    c = PagedCache.empty(2, 16, 1, 16, device=DEV)
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    step = PagedStep.of([(0, 5, [1]), (0, 0, [])], DEV)
    tree = PagedTree(step, none)
    assert tree.masks.shape == (0, 1)
    assert c.attend(torch.zeros(0, 1, 16, dtype=BF, device=DEV), step, tree=tree).shape == (0, 1, 16)
    kept, counts, following = tree.accept(torch.zeros(0, 50, device=DEV), none)
    assert kept.shape == (0,) and counts.tolist() == [0, 0] and following.tolist() == [-1, -1]
    PagedLayers([c]).keep(step, kept, counts)
    i = lambda *shape: torch.zeros(*shape, dtype=torch.int32, device=DEV)  # noqa: E731
    step = PagedStep(i(1), i(0), i(0, 4), rows=3)
    tree = PagedTree(step, torch.full((3,), -1, dtype=torch.int32, device=DEV))
    assert not tree.masks.any() and not tree.positions.any()
    assert not c.attend(torch.ones(3, 1, 16, dtype=BF, device=DEV), step, tree=tree).any()
    kept, counts, following = tree.accept(torch.zeros(3, 50, device=DEV), i(3))
    assert kept.tolist() == [-1] * 3 and counts.shape == (0,)
    PagedLayers([c]).keep(step, kept, counts)


def test_refusals_on_the_device():
    from lit_llama_b200 import PagedCache, PagedLayers, PagedStep, PagedTree

    c = PagedCache.empty(2, 16, 1, 16, device=DEV)
    step = PagedStep.of([(3, 5, [1])], DEV)
    parents = torch.tensor([-1, 0, 1], dtype=torch.int32, device=DEV)
    tree, other = PagedTree(step, parents), PagedTree(PagedStep.of([(3, 5, [1])], DEV), parents)
    q = torch.zeros(3, 1, 16, dtype=BF, device=DEV)
    with pytest.raises(ValueError, match="another step"):
        c.attend(q, step, tree=other)
    for bad in (parents.long(), parents[:2], parents.cpu(), torch.zeros(6, dtype=torch.int32, device=DEV)[::2], parents[None]):
        with pytest.raises(ValueError):
            PagedTree(step, bad)
    x, tokens = torch.zeros(3, 50, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    for kw in (dict(logits=x[:2]), dict(logits=x.double()), dict(logits=x[0]), dict(logits=x.cpu()), dict(tokens=tokens.float()), dict(tokens=tokens[:2]), dict(temperature=-1.0),
               dict(temperature=float("nan")), dict(temperature=1.0, noise=x[:, :49]), dict(temperature=1.0, noise=x.to(BF)), dict(temperature=float("inf"))):
        with pytest.raises(ValueError):
            tree.accept(**dict(dict(logits=x, tokens=tokens), **kw))
    layers, n = PagedLayers([c]), torch.ones(1, dtype=torch.int32, device=DEV)
    for kept, counts in ((parents.long(), n), (parents[:2], n), (parents, n[:0]), (parents, n.cpu())):
        with pytest.raises(ValueError):
            layers.keep(step, kept, counts)
    for pairs in (torch.zeros(2, 2, device=DEV), torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 4, dtype=torch.int32, device=DEV)[:, ::2]):
        with pytest.raises(ValueError):
            layers.copy(pairs)
