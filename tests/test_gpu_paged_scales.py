"""GPU: scales that a row must not depend on: those of pages that are not there."""
import math

import pytest
import torch

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
