"""GPU: scales that a row must not depend on: those of pages that are not there."""
import math

import pytest
import torch

import paged_oracle as O
from test_gpu_paged import DEV, IDS, TYPES, check, gen, make

pytestmark = pytest.mark.gpu

CODES = [t for t in TYPES if t[1] != "act"]


@pytest.mark.parametrize("dtype,store", CODES, ids=[i for t, i in zip(TYPES, IDS) if t[1] != "act"])
@pytest.mark.parametrize("sequences,lost,window,first", [
    ([(70, 200), (100, 300)], [0, 1, 2], 0, 0),             # the first pages of every sequence
    ([(90, 150)], [3, 8], 0, 0),
    ([(1, 200), (1, 90)], [0, 3], 0, 0),
    ([(200, 900)], list(range(1, 30)), 300, 5),             # what lies behind a window
])
def test_pages_that_are_not_there_bring_no_scales(dtype, store, sequences, lost, window, first):
    """The first place of the pool, which belongs to none of the sequences here, has scales of any size: the results are the same to the last bit."""
    from lit_llama_b200 import PagedStep

    cache, _, seqs = make(dtype, store, 2, 64, 64, 16, sequences, spare=8)
    free = set(range(cache.n_pages)) - {p for _, _, pages in seqs for p in pages}
    if 0 not in free:                                       # page 0 is nobody's
        other = min(free)
        seqs = [(n, m, [other if p == 0 else p for p in pages]) for n, m, pages in seqs]
    seqs = [(n, m, [-1 if i in lost else p for i, p in enumerate(pages)]) for n, m, pages in seqs]
    step = PagedStep.of(seqs, DEV)
    q = torch.randn(step.rows, 8, 64, generator=gen(4)).to(dtype)
    results = []
    for scale in (1.0, 2.0 ** 30, 2.0 ** -30, 0.0, math.inf, math.nan):
        for t in (cache.k_scale, cache.v_scale):
            t[0] = scale
        results.append(cache.attend(q.to(DEV), step, window=window, first=first))
    check(results[0], q, cache, seqs, 0.125, window, first)
    assert all(torch.equal(r, results[0]) for r in results[1:])


@pytest.mark.parametrize("dtype,store", CODES, ids=[i for t, i in zip(TYPES, IDS) if t[1] != "act"])
@pytest.mark.parametrize("sequences,window,first", [([(200, 900)], 300, 5), ([(90, 333), (40, 200)], 64, 0), ([(1, 300), (1, 90)], 50, 3)])
def test_keys_before_every_window_bring_no_scales(dtype, store, sequences, window, first):
    cache, step, seqs = make(dtype, store, 2, 64, 64, 16, sequences)
    q = torch.randn(step.rows, 8, 64, generator=gen(4)).to(dtype)
    results = []
    for scale in (1.0, 2.0 ** 30, 2.0 ** -30, 0.0, math.inf, math.nan):
        for new, length, pages in seqs:
            for j in range(first, length - new - window + 1):
                for t in (cache.k_scale, cache.v_scale):
                    t[pages[j // 16], :, j % 16] = scale
        results.append(cache.attend(q.to(DEV), step, window=window, first=first))
    check(results[0], q, cache, seqs, 0.125, window, first)
    assert all(torch.equal(r, results[0]) for r in results[1:])


@pytest.mark.parametrize("store", ["fp8", "int8"])
@pytest.mark.parametrize("sequences", [[(90, 700)], [(120, 500), (1, 300), (40, 40)]])
@pytest.mark.parametrize("where,exponent", [("early", -20), ("early", -14), ("early", 9), ("early", 15), ("early", 30), ("late", 9), ("late", 30), ("late", 70), ("rising", 1), ("falling", 1),
                                            ("most", -13), ("most", -30), ("none", 0)])
def test_scales_far_from_the_others(store, sequences, where, exponent):
    """Values, keys and both whose scales are far from the others' at one place, at most places, or rise and fall along the sequence."""
    for which in ("k", "v", "kv"):
        cache, step, seqs = make(torch.bfloat16, store, 2, 64, 32, 16, sequences)
        for name in which:
            t = cache.k_scale if name == "k" else cache.v_scale
            by = 2.0 ** (exponent / 4 if name == "k" and exponent > 0 and where in ("early", "late") else exponent)      # (a key's makes its scores large)
            for new, length, pages in seqs:
                for j in range(length):
                    at = (pages[j // 16], slice(None), j % 16)
                    if where == "early" and j == 3 or where == "late" and j == length - new // 2 - 1 or where == "most" and j >= 5:
                        t[at] *= by
                    elif where in ("rising", "falling"):
                        t[at] *= 2.0 ** ((j if where == "rising" else length - j) * (4 if name == "k" else 40) / length - (4 if name == "k" else 20))
                    elif where == "none" and j < 140:
                        t[at] = 0.0
        q = torch.randn(step.rows, 8, 64, generator=gen(4)).to(torch.bfloat16)
        got = cache.attend(q.to(DEV), step)
        want, mag, dots = O.attend(q, cache, seqs, 0.125)
        # Beside the roundings relative to each entry (weights, codes times scales, outputs):
        #   a small scale's factor is off by 2^-25 where the largest of the sequence, which a row need not see, is 1 .. 2: c 2^-25 for an entry (c the largest code) and
        #   2^-24 for two roundings of a product below f16's normal numbers; a row whose largest output is so small that this is more than 2^-12 of it is computed in f32
        #   the same of keys changes a score by up to 2^-10, and so does its reference; else the row is computed in f32
        #   weights are in f16, the largest at least 2^6, so each is off by half the least step, 2^-25, whatever its size: 2^-31 of the sum of the values' absolute values
        c = O.LARGEST[store]

        def seen(x):                                                             # [pages, heads, page, ..] of each row's keys, one after the other
            return [torch.cat(list(x.cpu()[torch.tensor(pages)].transpose(1, 2)))[:length].double() for _, length, pages in seqs]

        largest = torch.cat([x.amax(0).expand(new, 2) for x, (new, _, _) in zip(seen(cache.v_scale), seqs)]).repeat_interleave(4, 1)[..., None]
        total = torch.cat([x.abs().cumsum(0)[length - new:] for x, (new, length, _) in zip(seen(O.values(cache, "v")), seqs)]).repeat_interleave(4, 1)
        peak = want.abs().amax(-1, keepdim=True)
        tol = O.tolerance(want, mag, dots, 64, 700, False, store) + torch.minimum((c * 2.0 ** -25 + 2.0 ** -24) * largest, 2.0 ** -12 * peak) + 2.0 ** -31 * total
        tol = tol + ("k" in which) * 2 * 2.0 ** -10 * mag + 2.0 ** -133        # (and bf16's least step)
        off = (got.cpu().double() - want).abs()
        assert bool((off <= tol).all()), (which, float((off / tol).max()))


@pytest.mark.parametrize("store", ["fp8", "int8"])
def test_far_scales_of_one_sequence_reach_no_other(store):
    """Some hundred short sequences, several row tiles for every SM; every third has scales far below its others, and scores so large that this matters.  The same
    bits every time, and those of the others whether or not it has."""
    sequences = [(5 + i % 30, 40 + 7 * (i % 50)) for i in range(300)]
    cache, step, seqs = make(torch.bfloat16, store, 8, 32, 32, 16, sequences)
    q = (torch.randn(step.rows, 8, 32, generator=gen(4)) * 200).to(torch.bfloat16).to(DEV)
    others = torch.cat([torch.full((n,), i % 3 != 1) for i, (n, _, _) in enumerate(seqs)])
    usual = cache.attend(q, step)
    for i in range(1, 300, 3):
        for t in (cache.k_scale, cache.v_scale):
            t[seqs[i][2][1]] *= 2.0 ** -14
    first = cache.attend(q, step)
    assert torch.equal(first.cpu()[others], usual.cpu()[others]) and not torch.equal(first, usual)
    for _ in range(10):
        assert torch.equal(cache.attend(q, step), first)
