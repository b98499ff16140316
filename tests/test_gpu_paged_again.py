"""GPU: rows that are computed again, because a result is not finite or a scale is out of range: infinities and NaN in single entries, some rows of a tile and not
others, behind windows, beside pages that are not there, in every form of the kernels."""
import math

import pytest
import torch

import paged_oracle as O
from test_gpu_paged import DEV, IDS, TYPES, gen, make

pytestmark = pytest.mark.gpu

FORMS = [                                                   # heads, kv heads, K, V, page, sequences, window, first
    (8, 2, 64, 48, 16, [(1, 100), (1, 33), (1, 70)], 0, 0),
    (8, 2, 64, 48, 16, [(1, 300), (3, 77)], 40, 5),
    (4, 4, 128, 128, 64, [(1, 2500)], 0, 0),                # in parts
    (8, 2, 64, 48, 16, [(40, 100), (150, 150), (1, 80)], 0, 0),
    (8, 2, 64, 128, 32, [(90, 500)], 70, 3),
    (4, 1, 64, 64, 64, [(300, 2000)], 0, 0),                # row tiles cut among the SMs
    (6, 2, 256, 256, 16, [(20, 60), (1, 5)], 0, 0),
]


def expect(got, q, cache, seqs, scale, window, first):
    """Where the formula's result is finite it is that, elsewhere the same infinity or NaN."""
    want, mag, dots = O.attend(q, cache, seqs, scale, window, first)
    got = got.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[want.isinf()], want[want.isinf()]) and torch.isfinite(got[fine]).all()
    tol = O.tolerance(want, mag, dots, cache.dim, max(m for _, m, _ in seqs), q.dtype == torch.float32, cache.store)
    assert bool(((got - want).abs() <= tol)[fine].all())
    return fine


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "f32"])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_single_entries_that_are_not_finite(dtype, form):
    heads, G, K, V, page, sequences, window, first = FORMS[form]
    cache, step, seqs = make(dtype, "act", G, K, V, page, sequences)
    g = gen(9)
    for new, length, pages in seqs:                         # values: columns of some keys, early, late and among the new ones
        for n, bad in enumerate((math.inf, -math.inf, math.nan, math.inf, math.nan)):
            j = [0, length // 2, length - 1, length - (new + 1) // 2, max(length - new - 1, 0)][n]
            cache.v[pages[j // page], int(torch.randint(G, (1,), generator=g)), j % page, int(torch.randint(V, (1,), generator=g))] = bad
    q = torch.randn(step.rows, heads, K, generator=g).to(dtype)
    fine = expect(cache.attend(q.to(DEV), step, window=window, first=first), q, cache, seqs, K ** -0.5, window, first)
    assert fine.any() and not fine.all()
    for new, length, pages in seqs:                         # a key: its score is NaN, and with it all of the rows that see it
        j = length - (new + 1) // 2
        cache.k[pages[j // page], 0, j % page, 3] = math.nan
    fine = expect(cache.attend(q.to(DEV), step, window=window, first=first), q, cache, seqs, K ** -0.5, window, first)
    assert fine.any()


@pytest.mark.parametrize("dtype,store", [t for t in TYPES if t[1] != "act"], ids=[i for t, i in zip(TYPES, IDS) if t[1] != "act"])
@pytest.mark.parametrize("form", range(len(FORMS)))
def test_scales_that_are_not_finite_or_out_of_range(dtype, store, form):
    from lit_llama_b200 import PagedStep

    heads, G, K, V, page, sequences, window, first = FORMS[form]
    cache, step, seqs = make(dtype, store, G, K, V, page, sequences)
    q = torch.randn(step.rows, heads, K, generator=gen(9)).to(dtype)
    seqs = [(n, m, [-1 if i == 1 and m - n > 3 * page else p for i, p in enumerate(pages)]) for n, m, pages in seqs]
    step = PagedStep.of(seqs, DEV)
    for new, length, pages in seqs:
        j = length - (new + 1) // 2
        cache.v_scale[pages[j // page], 0, j % page] = 2.0 ** 62
        cache.v_scale[pages[j // page], G - 1, j % page] = math.inf
    expect(cache.attend(q.to(DEV), step, window=window, first=first), q, cache, seqs, K ** -0.5, window, first)
    for new, length, pages in seqs:
        j = length - (new + 1) // 2
        cache.v_scale[pages[j // page], G - 1, j % page] = math.nan
        cache.k_scale[pages[j // page], 0, j % page] = math.nan
    fine = expect(cache.attend(q.to(DEV), step, window=window, first=first), q, cache, seqs, K ** -0.5, window, first)
    assert not fine.all()


def test_rows_that_take_long_hold_nobody_up():
    """Three row tiles of 256 rows for every SM, each over 24576 keys; the last 32 rows of each see a value whose scale is out of range.  One warp computes them again
    for longer than a wait lasted once; the others wait for it and go on as ever: their rows have the bits that they have without that scale."""
    from lit_llama_b200 import PagedCache, PagedStep

    heads, length, new, page = 3 * torch.cuda.get_device_properties(0).multi_processor_count, 24576, 256, 256
    n_pages = length // page
    g = torch.Generator(DEV).manual_seed(1)
    cache = PagedCache.empty(n_pages, page, heads, 16, 16, store="int8", device=DEV)
    for pool, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        pool.copy_((torch.randn(pool.shape, generator=g, device=DEV) * 60).round().clamp(-127, 127).to(torch.int8))
        scale.fill_(2.0 ** -6)
    step = PagedStep.of([(new, length, list(range(n_pages)))], DEV)
    q = torch.randn(new, heads, 16, generator=g, device=DEV).to(torch.bfloat16)
    usual = cache.attend(q, step)
    at = length - 32
    cache.v_scale[at // page, :, at % page] = 2.0 ** 70
    got = cache.attend(q, step)
    assert torch.equal(got[:224], usual[:224])
    for h in range(0, heads, 37):                           # and the others the formula's value: some heads, in 64 bits
        k, v = (x[:, h].double().reshape(length, 16) * s[:, h].double().reshape(length, 1) for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
        s = (q[224:, h].double() @ k.T * 0.25).masked_fill(torch.arange(length, device=DEV)[None] > torch.arange(at, length, device=DEV)[:, None], -math.inf)
        w = torch.softmax(s, -1)
        dots = (q[224:, h].double().abs() @ k.abs().T).amax(-1) * 0.25
        tol = O.tolerance(w @ v, w @ v.abs(), dots, 16, length, False, "int8")
        assert bool(((got[224:, h].double() - w @ v).abs() <= tol).all())
