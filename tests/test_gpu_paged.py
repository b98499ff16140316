"""GPU: paged caches against the plain restatement in tests/paged_oracle.py (64 bits): rows written and read back in every type, attention of single
tokens, chunks and both together over pages, windows with first tokens, pages that are not there, values that no row may see, strides, streams,
recorded steps, and a sequence served from its prompt on."""
import math

import pytest
import torch

import paged_oracle as O

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [(torch.bfloat16, "act"), (torch.bfloat16, "fp8"), (torch.bfloat16, "int8"), (torch.float32, "act"), (torch.float32, "fp8"), (torch.float32, "int8")]
IDS = ["bf16", "bf16-fp8", "bf16-int8", "f32", "f32-fp8", "f32-int8"]


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make(dtype, store, kv_heads, dim, vdim, page, sequences, seed=1, spare=2, std=1.0):
    """A cache whose sequences [(new, length)] are already there, and the step: (cache, step, [(new, length, pages)])."""
    from lit_llama_b200 import PagedCache, PagedStep

    g = gen(seed)
    n_pages = sum(-(-m // page) for _, m in sequences) + spare
    seqs = O.random_pages(sequences, page, n_pages, g)
    cache = PagedCache.empty(n_pages, page, kv_heads, dim, vdim, dtype=dtype, store=store, device=DEV)
    for pool, scale, mean in ((cache.k, cache.k_scale, 0.0), (cache.v, cache.v_scale, 0.3)):
        x = (torch.randn(pool.shape, generator=g) * std + mean).to(dtype)
        if store == "act":
            pool.copy_(x)
        else:
            code, s = O.quantise(x, store)
            pool.copy_(code.to(pool.dtype))
            scale.copy_(s)
    return cache, PagedStep.of(seqs, DEV), seqs


def check(got, q, cache, seqs, scale, window=0, first=0):
    want, mag, dots = O.attend(q, cache, seqs, scale, window, first)
    f32 = q.dtype == torch.float32
    keys = max(m for _, m, _ in seqs)
    tol = O.tolerance(want, mag, dots, cache.dim, keys, f32, cache.store)
    off = (got.cpu().double() - want).abs()
    assert bool((off <= tol).all()), (float((off / tol).max()), float(off.max()))
    assert O.rel(got, want) < (3e-6 if f32 else 2.0 ** -8), O.rel(got, want)


# ----------------------------------------------------------------------------- rows
@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
@pytest.mark.parametrize("kv_heads,dim,vdim,page,sequences", [
    (1, 16, 16, 16, [(1, 1)]),
    (8, 128, 128, 64, [(1, 40), (1, 1), (0, 7), (1, 129)]),
    (5, 80, 96, 16, [(7, 7), (33, 49), (0, 0), (1, 16), (40, 95)]),
    (2, 256, 240, 256, [(300, 300), (5, 517)]),
    (32, 192, 128, 32, [(70, 75)] + [(1, 3 + i) for i in range(40)]),
])
def test_rows_go_in_and_come_back(dtype, store, kv_heads, dim, vdim, page, sequences):
    cache, step, seqs = make(dtype, store, kv_heads, dim, vdim, page, sequences)
    rows, g = step.rows, gen(7)
    k, v = (torch.randn(rows, kv_heads, d, generator=g).to(dtype) for d in (dim, vdim))
    k[0] = 0.0                                                           # a row of zeros, tiny ones, one of huge spread
    if rows > 3:
        v[1], k[2] = v[1] * 1e-38, (k[2].float() * torch.logspace(-20, 20, dim)).to(dtype)
    want = {}
    for name, x in (("k", k), ("v", v)):
        pool, scale = getattr(cache, name).cpu().float(), getattr(cache, name + "_scale")
        scale = None if scale is None else scale.cpu()
        code, s = (x.float(), None) if store == "act" else O.quantise(x, store)
        for r, (_, _, pg, at) in enumerate(O.places(seqs, page)):
            pool[pg, :, at] = code[r]
            if s is not None:
                scale[pg, :, at] = s[r]
        want[name] = (pool, scale, code if s is None else code * s[..., None])
    cache.write(k.to(DEV), v.to(DEV), step)
    back = cache.read(step)
    for (name, got), b in zip((("k", cache.k), ("v", cache.v)), back):
        pool, scale, value = want[name]
        assert torch.equal(got.cpu().float(), pool)                        # and every other place as it was
        if scale is not None:
            assert torch.equal(getattr(cache, name + "_scale").cpu(), scale)
        assert torch.equal(b.cpu(), value.to(dtype))


@pytest.mark.parametrize("store", ["fp8", "int8"])
def test_codes_are_off_by_half_a_step(store):
    cache, step, seqs = make(torch.float32, store, 3, 64, 64, 16, [(50, 50)])
    x = torch.randn(50, 3, 64, generator=gen(3)) * torch.logspace(-6, 6, 50)[:, None, None]
    cache.write(x.to(DEV), x.to(DEV), step)
    back, _ = cache.read(step)
    top = x.abs().amax(-1, keepdim=True)
    half = top / 127 / 2 if store == "int8" else torch.maximum(x.abs() * 2.0 ** -4, top / 448 * 2.0 ** -10)      # e4m3: relative, or half the smallest subnormal
    assert bool(((back.cpu() - x).abs() <= half * (1 + 2.0 ** -20)).all())


@pytest.mark.parametrize("store", ["fp8", "int8"])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_row_with_an_infinity_reads_back_as_nan_and_its_codes_are_finite(store, bad):
    cache, step, seqs = make(torch.bfloat16, store, 2, 32, 48, 16, [(3, 3)])
    k, v = torch.ones(3, 2, 32, dtype=torch.bfloat16), torch.ones(3, 2, 48, dtype=torch.bfloat16)
    k[1, 0, 5] = bad
    v[2, 1, 47] = bad
    cache.write(k.to(DEV), v.to(DEV), step)
    bk, bv = (x.cpu() for x in cache.read(step))
    assert bk[1, 0].isnan().all() and bv[2, 1].isnan().all() and bk.isnan().sum() == 32 and bv.isnan().sum() == 48
    assert torch.isfinite(cache.k.float()).all() and torch.isfinite(cache.v.float()).all()


@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
def test_rows_of_any_stride_and_rows_that_are_not_the_steps(dtype, store):
    """A slice of one product, a transposed one, rows off their 16-byte borders; rows behind the last sequence; pages that are not there."""
    from lit_llama_b200 import PagedStep

    cache, step, seqs = make(dtype, store, 4, 32, 16, 16, [(5, 20), (2, 2)])
    other, _, _ = make(dtype, store, 4, 32, 16, 16, [(5, 20), (2, 2)])
    wide = torch.randn(9, 4 * 100 + 3, generator=gen(2)).to(dtype).to(DEV)
    k, v = wide[:, :128].view(9, 4, 32), wide[:, 200:264].view(9, 4, 16)
    cache.write(k, v, step)                                              # 9 rows, the step has 7
    for a, b in ((k.transpose(0, 1).contiguous().transpose(0, 1), v.transpose(1, 2).contiguous().transpose(1, 2)),
                 (wide[:, 1:129].clone().view(9, 4, 32), torch.cat([wide[:, :1], v.reshape(9, 64)], 1)[:, 1:].unflatten(1, (4, 16)))):
        a = k if not torch.equal(a, k) else a
        other.write(a, b, step)
        for x, y in ((cache.k, other.k), (cache.v, other.v)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))
    before = [t.clone() for t in (cache.k, cache.v)]
    for page in (-1, cache.n_pages, 2 ** 31 - 1, -2 ** 31):
        s = PagedStep.of([(5, 20, [seqs[0][2][0], page])], DEV)
        cache.write(k, v, s)                                             # 4 rows on the page that is not there
        bk, bv = cache.read(s)
        assert (bk[1:] == 0).all() and (bv[1:] == 0).all()
    before[0][seqs[0][2][0]], before[1][seqs[0][2][0]] = cache.k[seqs[0][2][0]], cache.v[seqs[0][2][0]]
    assert torch.equal(before[0].view(torch.uint8), cache.k.view(torch.uint8)) and torch.equal(before[1].view(torch.uint8), cache.v.view(torch.uint8))


# ----------------------------------------------------------------------------- attention
SHAPES = [
    # heads, kv_heads, dim, vdim, page, sequences
    (1, 1, 16, 16, 16, [(1, 1)]),
    (4, 4, 128, 128, 64, [(1, n) for n in (1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 200)]),
    (32, 8, 128, 128, 16, [(1, 700), (0, 5), (1, 1), (1, 1030)]),
    (16, 1, 64, 128, 32, [(1, 333), (1, 48)]),
    (40, 2, 64, 64, 32, [(1, 77), (2, 90)]),                               # 20 heads a group: a token's rows fill more than one tile
    (6, 2, 80, 48, 16, [(7, 7), (30, 81), (1, 50)]),
    (6, 2, 96, 112, 64, [(129, 129), (0, 0), (3, 500), (1, 1), (64, 64)]),
    (8, 2, 128, 128, 128, [(200, 777)]),
    (4, 2, 192, 128, 16, [(45, 45), (1, 300), (150, 170)]),
    (4, 4, 256, 256, 64, [(1, 100), (20, 130)]),
    (2, 1, 16, 240, 16, [(33, 40)]),
]


@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
@pytest.mark.parametrize("shape", SHAPES, ids=[str(i) for i in range(len(SHAPES))])
def test_attention(dtype, store, shape):
    heads, kv_heads, dim, vdim, page, sequences = shape
    cache, step, seqs = make(dtype, store, kv_heads, dim, vdim, page, sequences)
    q = torch.randn(step.rows, heads, dim, generator=gen(5)).to(dtype)
    got = cache.attend(q.to(DEV), step)
    assert got.dtype == dtype and got.shape == (step.rows, heads, vdim)
    check(got, q, cache, seqs, dim ** -0.5)


@pytest.mark.parametrize("dtype,store", [TYPES[0], TYPES[2], TYPES[3]], ids=[IDS[0], IDS[2], IDS[3]])
@pytest.mark.parametrize("window,first", [(1, 0), (1, 1), (16, 0), (17, 3), (64, 16), (100, 130), (500, 4), (4000, 40), (130, 1000)])
def test_windows_and_first_tokens(dtype, store, window, first):
    for page, sequences in ((16, [(1, 1), (1, 130), (1, 400), (1, 16), (1, 17)]), (64, [(90, 90), (40, 333), (1, 250), (140, 460)])):
        cache, step, seqs = make(dtype, store, 2, 64, 64, page, sequences, seed=window)
        q = torch.randn(step.rows, 8, 64, generator=gen(6)).to(dtype)
        check(cache.attend(q.to(DEV), step, scale=0.2, window=window, first=first), q, cache, seqs, 0.2, window, first)


@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
def test_a_long_sequence_in_parts(dtype, store):
    """One token, and few, of a sequence long enough for its keys to be shared among CTAs; peaked scores, so one part has nearly all the weight."""
    for new, heads in ((1, 4), (4, 4), (1, 1)):
        cache, step, seqs = make(dtype, store, 1, 64, 32, 16, [(new, 9001)], std=1.0)
        q = torch.randn(new, heads, 64, generator=gen(8)).to(dtype) * 2
        check(cache.attend(q.to(DEV), step), q, cache, seqs, 0.125)
        check(cache.attend(q.to(DEV), step, window=6000, first=100), q, cache, seqs, 0.125, 6000, 100)


@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
def test_a_chunk_over_a_long_sequence(dtype, store):
    cache, step, seqs = make(dtype, store, 2, 128, 128, 64, [(60, 4500), (1, 4000)])
    q = torch.randn(step.rows, 8, 128, generator=gen(9)).to(dtype)
    check(cache.attend(q.to(DEV), step), q, cache, seqs, 128 ** -0.5)


SHARES = [                                          # heads, kv heads, K, V, page, window, first, sequences: row tiles of 256 rows cut among the SMs
    (4, 1, 64, 64, 64, 0, 0, [(700, 20000)]),                              # each over many SMs
    (8, 2, 64, 64, 32, 0, 0, [(1, 9000), (300, 300), (1, 1), (0, 50), (513, 4000), (1, 5000), (65, 65)]),      # single tokens among chunks
    (8, 8, 32, 32, 16, 0, 0, [(5 + i % 30, 5 + 7 * i) for i in range(150)]),      # more row tiles than SMs, short ones
    (64, 1, 128, 64, 16, 0, 0, [(9, 700), (130, 500)]),                    # a group of 64 heads
    (4, 2, 192, 128, 128, 200, 3, [(400, 6000), (1, 6000), (600, 600)]),   # windows: few keys for each
    (12, 4, 64, 64, 64, 0, 0, [(1 + i % 4, 9000 - 100 * i) for i in range(60)] + [(200, 300), (0, 7), (9, 9), (1, 1)]),      # both kernels: 8 packed rows and more
    (16, 1, 64, 64, 64, 0, 0, [(1, 9000 - 60 * i) for i in range(100)] + [(64, 3000), (2, 70)]),      # and 16
]


@pytest.mark.parametrize("dtype,store", TYPES[:3], ids=IDS[:3])
@pytest.mark.parametrize("shape", SHARES, ids=[str(i) for i in range(len(SHARES))])
def test_row_tiles_shared_among_sms(dtype, store, shape):
    heads, kv_heads, dim, vdim, page, window, first, sequences = shape
    cache, step, seqs = make(dtype, store, kv_heads, dim, vdim, page, sequences)
    q = torch.randn(step.rows, heads, dim, generator=gen(3)).to(dtype)
    check(cache.attend(q.to(DEV), step, window=window, first=first), q, cache, seqs, dim ** -0.5, window, first)


@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
def test_sequences_shorter_than_their_new_tokens(dtype, store):
    """Lengths that were changed on the device: rows at negative positions see nothing, the others what there is."""
    cache, step, seqs = make(dtype, store, 2, 64, 64, 16, [(40, 40), (300, 300), (1, 1), (200, 900)])
    lengths = [7, 10, 0, 100]
    step.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    seqs = [(n, m, pages) for (n, _, pages), m in zip(seqs, lengths)]
    q = torch.randn(step.rows, 8, 64, generator=gen(3)).to(dtype)
    got = cache.attend(q.to(DEV), step)
    check(got, q, cache, seqs, 0.125)
    assert not got[:33].any() and not got[40:330].any() and not got[340].any() and not got[341:441].any()


@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
def test_pages_that_are_not_there(dtype, store):
    """Keys on them are not seen, whatever is in the pool; a row that sees nothing attends to zeros."""
    from lit_llama_b200 import PagedStep

    cache, _, seqs = make(dtype, store, 2, 64, 64, 16, [(1, 200), (50, 120), (1, 20), (130, 140)])
    lost = []
    for i, (new, length, pages) in enumerate(seqs):
        pages = list(pages)
        for j, x in ((2, -1), (3, cache.n_pages), (5, 2 ** 31 - 1), (0, -2 ** 31)):
            if j < len(pages) and i != 2:
                pages[j] = x
        if i == 2:
            pages = [-1] * len(pages)
        lost.append((new, length, pages))
    step = PagedStep.of(lost, DEV)
    q = torch.randn(step.rows, 4, 64, generator=gen(4)).to(dtype)
    got = cache.attend(q.to(DEV), step)
    check(got, q, cache, lost, 0.125)
    assert (got[51] == 0).all() and (got[52:58] == 0).all()
    # positions below zero (lengths that are shorter than the new tokens), a table that is too short
    starts, lengths = torch.tensor([0, 5, 9], dtype=torch.int32, device=DEV), torch.tensor([3, 1000], dtype=torch.int32, device=DEV)
    s = PagedStep(starts, lengths, torch.tensor([[0, 1], [2, 3]], dtype=torch.int32, device=DEV), rows=9)
    got = cache.attend(q[:9].to(DEV), s)
    assert (got[:2] == 0).all()
    check(got[2:], q[2:9], cache, [(3, 3, [0, 1]), (4, 32, [2, 3])], 0.125)


@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_what_no_row_may_see(dtype, store, bad):
    """Infinities and NaN in unused pages, behind the last token, before the window and, for earlier rows of a chunk, in later tokens."""
    for sequences, window, first in (([(1, 100), (1, 33)], 0, 0), ([(1, 100), (1, 77)], 20, 3), ([(40, 100), (150, 150)], 0, 0), ([(70, 150)], 30, 2), ([(1, 5000)], 0, 0)):
        cache, step, seqs = make(dtype, store, 2, 64, 32, 16, sequences)
        rows, q = step.rows, torch.randn(step.rows, 4, 64, generator=gen(4)).to(dtype)
        hurt = [t for t in ((cache.k, cache.v) if store == "act" else (cache.k_scale, cache.v_scale))]
        used = {p for _, _, pages in seqs for p in pages}
        for t in hurt:
            for p in set(range(cache.n_pages)) - used:
                t[p] = bad
            for new, length, pages in seqs:
                if length % 16:
                    t[pages[-1], :, length % 16:] = bad
                if window:
                    for j in range(first, length - new - window + 1):
                        t[pages[j // 16], :, j % 16] = bad
        got = cache.attend(q.to(DEV), step, window=window, first=first)
        assert torch.isfinite(got).all()
        check(got, q, cache, seqs, 0.125, window, first)
        # the last token of every sequence: only its own row sees it
        last = [sum(n for n, _, _ in seqs[:b + 1]) - 1 for b in range(len(seqs))]
        for new, length, pages in seqs:
            for t in hurt[1:]:
                t[pages[-1], :, (length - 1) % 16] = bad
        got = cache.attend(q.to(DEV), step, window=window, first=first).cpu()
        rest = [r for r in range(rows) if r not in last]
        want, mag, dots = O.attend(q, cache, seqs, 0.125, window, first)
        assert torch.isfinite(got[rest]).all() and not torch.isfinite(got[last]).any()
        assert torch.equal(got[last].isnan(), want[last].to(dtype).isnan())
        tol = O.tolerance(want, mag, dots, 64, 5000, dtype == torch.float32, store)
        assert bool(((got.double() - want).abs() <= tol)[rest].all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scores_of_any_size(dtype):
    """Infinite scores, scores of the type's lowest value, scores that all overflow downwards: the formula's result, or zeros where all weights are zero."""
    cache, step, seqs = make(dtype, "act", 1, 16, 16, 16, [(1, 40), (20, 40), (1, 40)])
    q = torch.zeros(step.rows, 2, 16, dtype=dtype)
    q[:, :, 0] = 1.0
    lowest = torch.finfo(dtype).min
    for b, value in ((0, lowest), (1, -math.inf), (2, math.inf)):
        for j in range(0, 40, 2):
            cache.k[seqs[b][2][j // 16], 0, j % 16, 0] = value
    got = cache.attend(q.to(DEV), step).cpu()
    want, mag, dots = O.attend(q, cache, seqs, 0.25)
    assert torch.isfinite(got[:21]).all() and got[21].isnan().all() and want[21].isnan().all()
    dots = torch.full_like(dots, 20.0)                                    # of the keys that count
    assert bool(((got.double() - want).abs() <= O.tolerance(want, mag, dots, 16, 40, dtype == torch.float32, "act"))[:21].all())
    for j in range(40):
        cache.k[seqs[0][2][j // 16], 0, j % 16, 0] = -math.inf
    assert (cache.attend(q.to(DEV), step)[0] == 0).all()


@pytest.mark.parametrize("dtype,store", [TYPES[0], TYPES[1], TYPES[5]], ids=[IDS[0], IDS[1], IDS[5]])
def test_queries_of_any_stride_and_rows_behind_the_last_sequence(dtype, store):
    cache, step, seqs = make(dtype, store, 2, 32, 32, 16, [(1, 30), (6, 50), (40, 60)])
    wide = torch.randn(step.rows + 4, 4 * 32 + 72, generator=gen(2)).to(dtype).to(DEV)
    q = wide[:, :128].view(-1, 4, 32)
    out = torch.full((step.rows + 4, 4, 32), 7.0, dtype=dtype, device=DEV)
    got = cache.attend(q, step, out=out)
    assert got is out and (out[step.rows:] == 7.0).all()
    check(out[:step.rows], q[:step.rows].cpu(), cache, seqs, 32 ** -0.5)
    assert torch.equal(cache.attend(q, step)[:step.rows], out[:step.rows]) and (cache.attend(q, step)[step.rows:] == 0).all()
    for same in (q.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([wide[:, :1], wide[:, :128]], 1)[:, 1:].unflatten(1, (4, 32)), q.transpose(1, 2).contiguous().transpose(1, 2)):
        assert torch.equal(cache.attend(same, step)[:step.rows], out[:step.rows])


@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
def test_what_the_host_says_of_a_step_changes_no_result(dtype, store):
    """Wrong numbers for the most new tokens and the longest sequence: other forms, the same sequences."""
    from lit_llama_b200 import PagedStep

    cache, step, seqs = make(dtype, store, 2, 64, 64, 32, [(1, 700), (130, 400), (3, 3), (40, 900)])
    q = torch.randn(step.rows, 8, 64, generator=gen(3)).to(dtype)
    for hints in (dict(), dict(max_new=1, max_length=16), dict(max_new=100000, max_length=10 ** 6), dict(max_new=1, max_length=900), dict(max_new=130)):
        s = PagedStep(step.starts, step.lengths, step.table, rows=step.rows, **hints)
        check(cache.attend(q.to(DEV), s), q, cache, seqs, 0.125)
    # no more rows than sequences, all of one of them
    cache, step, seqs = make(dtype, store, 2, 64, 64, 32, [(0, 5)] * 20 + [(40, 300)] + [(0, 0)] * 20)
    q = torch.randn(step.rows, 8, 64, generator=gen(3)).to(dtype)
    for hints in (dict(), dict(max_new=40)):
        check(cache.attend(q.to(DEV), PagedStep(step.starts, step.lengths, step.table, rows=step.rows, **hints)), q, cache, seqs, 0.125)


def test_the_same_call_gives_the_same_bits():
    for dtype, store in TYPES:
        cache, step, seqs = make(dtype, store, 2, 128, 128, 64, [(1, 3000), (100, 1000), (1, 5)])
        q = torch.randn(step.rows, 8, 128, generator=gen(3)).to(dtype).to(DEV)
        a = cache.attend(q, step)
        for _ in range(3):
            assert torch.equal(a, cache.attend(q, step))


def test_pools_beyond_32_bit_offsets():
    """Pages whose entries lie beyond 2^31 (of keys and of values) are written, read and attended to."""
    from lit_llama_b200 import PagedCache, PagedStep

    n_pages = (1 << 31) // (8 * 64 * 64) + 40
    for store in ("int8", "act"):
        cache = PagedCache.empty(n_pages, 64, 8, 64, dtype=torch.bfloat16, store=store, device=DEV)
        seqs = [(130, 130, [n_pages - 1, n_pages - 3, n_pages - 2]), (1, 64, [n_pages - 9])]
        step = PagedStep.of(seqs, DEV)
        g = gen(5)
        k, v, q = (torch.randn(131, h, 64, generator=g).to(torch.bfloat16) for h in (8, 8, 16))
        cache.write(k.to(DEV), v.to(DEV), step)
        bk, bv = cache.read(step)
        if store == "act":
            assert torch.equal(bk.cpu(), k) and torch.equal(bv.cpu(), v)
        got = cache.attend(q.to(DEV), step)
        small = PagedCache(*[None if t is None else t[-16:].clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)], dtype=torch.bfloat16)
        shifted = [(a, b, [p - n_pages + 16 for p in pages]) for a, b, pages in seqs]
        assert torch.equal(got, small.attend(q.to(DEV), PagedStep.of(shifted, DEV)))
        check(got, q, small, shifted, 0.125)
        del cache


@pytest.mark.parametrize("dtype,store", [t for t in TYPES if t[1] != "act"], ids=[i for t, i in zip(TYPES, IDS) if t[1] != "act"])
def test_places_never_written_count_as_zeros(dtype, store):
    """A pool begins as zeros with scales of zero: a row that sees such places weighs them with its score of zero, in units of their own and beside others."""
    cache, step, seqs = make(dtype, store, 2, 64, 64, 16, [(1, 64), (20, 100), (1, 40)])
    for _, length, pages in seqs:
        for p in pages[:1] + pages[2:3]:
            for t in (cache.k, cache.v):
                t.view(torch.uint8)[p, :, 3:] = 0
            for t in (cache.k_scale, cache.v_scale):
                t[p, :, 3:] = 0
    q = torch.randn(step.rows, 4, 64, generator=gen(4)).to(dtype)
    check(cache.attend(q.to(DEV), step), q, cache, seqs, 0.125)


@pytest.mark.parametrize("dtype,store", [t for t in TYPES if t[1] != "act"], ids=[i for t, i in zip(TYPES, IDS) if t[1] != "act"])
@pytest.mark.parametrize("low,high", [(-126, -100), (-24, -8), (-10, -7)])
def test_scales_of_keys_of_any_size(dtype, store, low, high):
    """Keys whose scales are powers of two, within what their codes in f16 take and far outside of it."""
    cache, step, seqs = make(dtype, store, 2, 64, 64, 16, [(1, 70), (20, 300), (1, 1), (90, 90)])
    exponents = torch.randint(low, high + 1, cache.k_scale.shape, generator=gen(3))
    cache.k_scale.copy_(torch.ldexp(torch.ones_like(exponents, dtype=torch.float64), exponents).float())
    q = torch.randn(step.rows, 4, 64, generator=gen(4)).to(dtype)
    check(cache.attend(q.to(DEV), step), q, cache, seqs, 0.125)


@pytest.mark.parametrize("dtype,store", [t for t in TYPES if t[1] != "act"], ids=[i for t, i in zip(TYPES, IDS) if t[1] != "act"])
@pytest.mark.parametrize("low,high", [(-126, -120), (-126, 0), (-100, -50), (-95, 90), (-70, 39), (30, 110)])
def test_scales_of_any_size(dtype, store, low, high):
    """Values whose scales are powers of two from one end of f32 to the other, small ones beside large ones."""
    cache, step, seqs = make(dtype, store, 2, 64, 64, 16, [(1, 70), (20, 100), (1, 1)])
    exponents = torch.randint(low, high + 1, cache.v_scale.shape, generator=gen(3))
    cache.v_scale.copy_(torch.ldexp(torch.ones_like(exponents, dtype=torch.float64), exponents).float())
    q = torch.randn(step.rows, 4, 64, generator=gen(4)).to(dtype)
    got = cache.attend(q.to(DEV), step)
    want, mag, dots = O.attend(q, cache, seqs, 0.125)
    tol = O.tolerance(want, mag, dots, 64, 100, dtype == torch.float32, store)
    # a score with the scale's logarithm is rounded at up to 128 (2^-18), and the logarithm is off by 2^-22 of up to 64
    # a small value beside large ones in f16: half its least step, 2^-25, where the largest scale is 1 .. 2
    if dtype == torch.bfloat16:
        tol += 2.0 ** -24 * float(cache.v_scale.max())
    tol += 2.0 ** -15 * mag + 2.0 ** -126 + want.abs() * (want.abs() < 2.0 ** -118)      # subnormal results
    assert bool(((got.cpu().double() - want).abs() <= tol).all())


# ----------------------------------------------------------------------------- streams, graphs, runs
@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
def test_a_recorded_step_follows_its_tensors(dtype, store):
    """A recorded write and attention of single tokens, replayed while the sequences grow; two recordings that take turns on two streams."""
    from lit_llama_b200 import PagedCache, PagedStep, PagePool

    heads, G, D, page = 4, 2, 64, 16
    made = []
    for which in range(2):
        pool = PagePool(400, page, DEV)
        cache = PagedCache.empty(400, page, G, D, dtype=dtype, store=store, device=DEV)
        first = pool.step([(b, 30 + 900 * b) for b in range(3)])
        g = gen(which)
        x = [torch.randn(first.rows, G, D, generator=g).to(dtype).to(DEV) for _ in range(2)]
        cache.write(*x, first)
        step = pool.step([(b, 1) for b in range(3)], width=150)
        q, k, v = (torch.zeros(3, h, D, dtype=dtype, device=DEV) for h in (heads, G, G))
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            cache.write(k, v, step)
            cache.attend(q, step)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                cache.write(k, v, step)
                out = cache.attend(q, step)
        torch.cuda.synchronize()
        made.append((pool, cache, step, q, k, v, graph, out, stream, g))
    for turn in range(4):
        for pool, cache, step, q, k, v, graph, out, stream, g in made:
            if turn:
                step.refill(pool.step([(b, 1) for b in range(3)]))
            for t in (q, k, v):
                t.copy_(torch.randn(t.shape, generator=g).to(dtype))
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for pool, cache, step, q, k, v, graph, out, stream, g in made:
            check(out, q.cpu(), cache, [(1, pool.position(b), pool.pages(b)) for b in range(3)], 0.125)


def test_calls_on_two_streams_at_once():
    cache, step, seqs = make(torch.bfloat16, "act", 2, 64, 64, 16, [(1, 5000), (200, 900), (1, 60)])
    q = [torch.randn(step.rows, 8, 64, generator=gen(i)).to(torch.bfloat16).to(DEV) for i in range(2)]
    alone = [cache.attend(x, step) for x in q]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(cache.attend(q[i], step))
    torch.cuda.synchronize()
    assert all(torch.equal(o, alone[i]) for i in range(2) for o in outs[i])


@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
@pytest.mark.parametrize("window,first", [(0, 0), (40, 5)])
def test_sequences_from_their_prompts_on(dtype, store, window, first):
    """Three requests served together: prompts in portions, then single tokens, pages booked as they grow and given back behind the window.  Every row
    attends to what was written (read back), at its own place in its sequence."""
    from lit_llama_b200 import PagedCache, PagePool

    heads, G, D, V, page = 6, 2, 64, 48, 16
    pool = PagePool(24, page, DEV, window=window, first=first)
    cache = PagedCache.empty(24, page, G, D, V, dtype=dtype, store=store, device=DEV)
    g = gen(11)
    total = {"a": 70, "b": 33, "c": 90}
    data = {r: [torch.randn(n + 8, h, d, generator=g).to(dtype) for h, d in ((heads, D), (G, D), (G, V))] for r, n in total.items()}
    kept = {r: ([], []) for r in total}                                    # keys and values as the pool has them
    plan = [[("a", 40), ("b", 33)], [("c", 64), ("a", 30), ("b", 1)], [("b", 1), ("c", 26)]] + [[("a", 1), ("b", 1), ("c", 1)]] * 6
    for entries in plan:
        at = {r: pool.position(r) if pool.has(r) else 0 for r, _ in entries}
        step = pool.step(entries)
        q, k, v = (torch.cat([data[r][i][at[r]:at[r] + n] for r, n in entries]).to(DEV) for i in range(3))
        cache.write(k, v, step)
        back = cache.read(step)
        got = cache.attend(q, step, window=window, first=first).cpu().double()
        row = 0
        for r, n in entries:
            for i in range(2):
                kept[r][i].append(back[i][row:row + n].cpu().double() if store == "act" else dequantised(cache, "kv"[i], pool, r, at[r], n))
            K, Vv = (torch.cat(x) for x in kept[r])
            for i in range(n):
                p = at[r] + i
                j = torch.tensor([x for x in range(p + 1) if not window or x > p - window or x < first])
                s = torch.einsum("hd,jhd->hj", data[r][0][p].double(), K[j].repeat_interleave(heads // G, 1)) * D ** -0.5
                want = torch.einsum("hj,jhd->hd", torch.softmax(s, 1), Vv[j].repeat_interleave(heads // G, 1))
                assert O.rel(got[row + i], want) < (3e-6 if dtype == torch.float32 else 2.0 ** -8)
            row += n
    for r in total:
        pool.release(r)
    assert pool.free_pages() == 24


def dequantised(cache, which, pool, request, at, n):
    x = O.values(cache, which)
    pages = pool.pages(request)
    return torch.stack([x[pages[p // cache.page], :, p % cache.page] for p in range(at, at + n)])
