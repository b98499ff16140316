"""CPU: paged caches without a device: what is refused, which pages a sequence has, and the arithmetic of units and splits that the kernels index by."""
import ctypes as C
import os
import random
import re

import pytest
import torch

import paged_oracle as O
from lit_llama_b200 import PagedCache, PagedStep, PagePool
from lit_llama_b200 import _seqlib as S
from lit_llama_b200 import paged
from lit_llama_b200.state import PoolFull

CPU = torch.device("cpu")


def pool(**kw):
    return PagePool(**dict(dict(n_pages=8, page=16, device=CPU), **kw))


# ----------------------------------------------------------------------------- pages
def test_pages_are_booked_as_sequences_grow_and_given_back():
    p = pool()
    s = p.step([("a", 17), ("b", 1)])
    assert s.rows == 18 and s.starts.tolist() == [0, 17, 18] and s.lengths.tolist() == [17, 1] and s.table.tolist() == [[0, 1], [2, -1]]
    assert (s.max_new, s.max_length) == (17, 17)
    s = p.step([("b", 15), ("a", 1)])
    assert s.lengths.tolist() == [16, 18] and s.table.tolist() == [[2, -1], [0, 1]] and p.position("a") == 18 and p.free_pages() == 5
    p.step([("b", 1)])
    assert p.pages("b") == [2, 3]
    p.release("a")
    assert not p.has("a") and p.free_pages() == 6
    assert p.step([("c", 33)]).table.tolist() == [[0, 1, 4]]


def test_a_step_that_does_not_fit_books_nothing():
    p = pool(n_pages=3)
    p.step([("a", 20)])
    with pytest.raises(PoolFull):
        p.step([("b", 5), ("a", 30)])
    assert not p.has("b") and p.position("a") == 20 and p.free_pages() == 1
    with pytest.raises(ValueError):
        p.step([("a", 1), ("a", 1)])
    with pytest.raises(ValueError):
        p.step([("a", -1)])
    assert p.position("a") == 20


@pytest.mark.parametrize("window,first", [(1, 0), (16, 0), (17, 3), (40, 16), (33, 17)])
def test_pages_behind_the_window_come_back_only_when_no_later_token_sees_them(window, first):
    p, page = pool(n_pages=12, window=window, first=first), 16
    length = 0
    for n in (1, 15, 1, 20, 3, 64, 1, 1, 30):
        p.step([("a", n)])
        for pos in range(length, length + n):                      # every key that a new row sees has its page
            for j in range(pos + 1):
                if j > pos - window or j < first:
                    assert p.pages("a")[j // page] >= 0, (pos, j)
        length += n
    held = [x for x in p.pages("a") if x >= 0]
    assert len(set(held)) == len(held) and p.free_pages() == 12 - len(held)
    assert len(held) <= -(-(window + 30) // page) + 1 + -(-first // page)
    p.release("a")
    assert p.free_pages() == 12


def test_empty_entries_and_widths():
    p = pool()
    s = p.step([("a", 0), ("b", 2)], width=5)
    assert s.rows == 2 and s.starts.tolist() == [0, 0, 2] and s.table.shape == (2, 5) and p.pages("a") == []
    s = p.step([])
    assert s.rows == 0 and s.seqs == 0
    t = PagedStep.of([(1, 3, [7])], CPU, width=3)
    u = PagedStep.of([(1, 20, [2, 5])], CPU)
    t.refill(u)
    assert t.lengths.tolist() == [20] and t.table.tolist() == [[2, 5, -1]]
    with pytest.raises(ValueError):
        u.refill(t)


@pytest.mark.parametrize("bad", [dict(n_pages=0), dict(page=8), dict(page=48), dict(window=-1), dict(first=-2)])
def test_pools_that_cannot_be(bad):
    with pytest.raises(ValueError):
        pool(**bad)


# ----------------------------------------------------------------------------- refusals
def cache(store="act", dtype=torch.bfloat16, **kw):
    return PagedCache.empty(**dict(dict(n_pages=4, page=16, kv_heads=2, dim=32, vdim=16, dtype=dtype, store=store, device="cpu"), **kw))


def test_the_kernels_run_on_cuda_only():
    c, s = cache(), PagedStep.of([(1, 1, [0])], CPU)
    k, v, q = torch.zeros(1, 2, 32, dtype=torch.bfloat16), torch.zeros(1, 2, 16, dtype=torch.bfloat16), torch.zeros(1, 4, 32, dtype=torch.bfloat16)
    for call in (lambda: c.write(k, v, s), lambda: c.read(s), lambda: c.attend(q, s)):
        with pytest.raises(RuntimeError, match="CUDA only"):
            call()


def test_pools_that_do_not_fit_are_refused():
    z = torch.zeros
    for store in ("fp8", "int8"):
        c = cache(store)
        assert c.bytes() == 4 * 2 * 16 * (32 + 16 + 8) and c.dtype == torch.bfloat16
        with pytest.raises(ValueError, match="scales"):
            PagedCache(c.k, c.v)
        with pytest.raises(ValueError, match="scales"):
            PagedCache(c.k, c.v, c.k_scale, c.v_scale[:2])
        with pytest.raises(ValueError, match="scales"):
            PagedCache(c.k, c.v, c.k_scale.half(), c.v_scale)
    c = cache()
    with pytest.raises(ValueError, match="belong together"):
        PagedCache(c.k, c.v.float())
    with pytest.raises(ValueError, match="belong together"):
        PagedCache(c.k, c.v[:2])
    with pytest.raises(ValueError, match="8-bit"):
        PagedCache(c.k, c.v, z(4, 2, 16), z(4, 2, 16))
    with pytest.raises(ValueError, match="contiguous"):
        PagedCache(c.k.transpose(0, 1), c.v.transpose(0, 1))
    with pytest.raises(ValueError, match="activations"):
        PagedCache(c.k, c.v, dtype=torch.float32)
    for bad in (dict(dim=24), dict(vdim=264), dict(dim=272), dict(page=20), dict(page=512), dict(kv_heads=0), dict(store="int4")):
        with pytest.raises(ValueError):
            cache(**bad)
    with pytest.raises(RuntimeError, match="float16"):
        cache(dtype=torch.float16)


def test_calls_that_do_not_fit_are_refused():
    c, s = cache(), PagedStep.of([(2, 2, [0])], CPU)
    q = torch.zeros(2, 4, 32, dtype=torch.bfloat16)
    for bad in (q[:, :3], q[:1], q.float(), q[:, :, :16], q[0]):
        with pytest.raises(ValueError):
            c.attend(bad, s)
    for kw in (dict(window=-1), dict(first=-1), dict(out=torch.zeros(2, 4, 32, dtype=torch.bfloat16)), dict(out=torch.zeros(2, 4, 16))):
        with pytest.raises(ValueError):
            c.attend(q, s, **kw)
    k, v = torch.zeros(2, 2, 32, dtype=torch.bfloat16), torch.zeros(2, 2, 16, dtype=torch.bfloat16)
    for a, b in ((k[:1], v), (k, v[:1]), (v, k), (k.float(), v), (k[:, :1], v)):
        with pytest.raises(ValueError):
            c.write(a, b, s)


def test_steps_that_do_not_fit_are_refused():
    i = lambda *shape: torch.zeros(*shape, dtype=torch.int32)  # noqa: E731
    PagedStep(i(3), i(2), i(2, 4), rows=5)
    for starts, lengths, table, rows in ((i(2), i(2), i(2, 4), 5), (i(3).long(), i(2), i(2, 4), 5), (i(3), i(2), i(3, 4), 5), (i(3), i(2), i(2, 0), 5), (i(3), i(2), i(4, 2).t(), 5),
                                         (i(3), i(2), i(2, 4), -1), (i(3), i(2), i(8), 5)):
        with pytest.raises(ValueError):
            PagedStep(starts, lengths, table, rows=rows)
    with pytest.raises(ValueError):
        PagedStep.of([(3, 2, [0])], CPU)


P8 = C.c_void_p(64)


def call(name, **kw):
    """A call of the C entry whose pointers are never followed: every one here is refused, or has nothing to do, before a launch."""
    lib = S.lib()
    base = dict(x=64, y=64, k=64, v=64, ks=None, vs=None, starts=64, lengths=64, table=64, ldt=4, width=4, rows=0, seqs=1, pages=4, page=16, heads=4, kv_heads=2, K=32, V=32, store=0, act=0,
                ld=64, hs=32, work=None, floats=0, window=0, first=0, scale=1.0)
    a = dict(base, **kw)
    if name == "attention":
        return lib.b2l_seq_paged_attention(a["x"], a["ld"], a["hs"], a["k"], a["v"], a["ks"], a["vs"], a["starts"], a["lengths"], a["table"], a["ldt"], a["width"], a["y"], a["work"],
                                           a["floats"], a["rows"], a["seqs"], a["pages"], a["page"], a["heads"], a["kv_heads"], a["K"], a["V"], a["window"], a["first"], a["scale"],
                                           0, 0, a["store"], a["act"], None)
    f = lib.b2l_seq_paged_write if name == "write" else lib.b2l_seq_paged_read
    return f(a["x"], a["ld"], a["hs"], a["y"], a["ld"], a["hs"], a["k"], a["v"], a["ks"], a["vs"], a["starts"], a["lengths"], a["table"], a["ldt"], a["width"], a["rows"], a["seqs"],
             a["pages"], a["page"], a["kv_heads"], a["K"], a["V"], a["store"], a["act"], None)


@pytest.mark.parametrize("name", ["write", "read", "attention"])
def test_the_c_entries_refuse_before_they_launch(name):
    assert call(name) == 0 and call(name, rows=5, seqs=0) == 0
    bad = [dict(x=None), dict(y=None), dict(k=None), dict(v=None), dict(starts=None), dict(lengths=None), dict(table=None), dict(store=1), dict(store=2, ks=64), dict(ldt=3), dict(width=0),
           dict(rows=-1), dict(seqs=-1), dict(pages=0), dict(page=24), dict(page=8), dict(page=512), dict(kv_heads=0), dict(K=24), dict(V=8), dict(K=272), dict(V=0), dict(store=3),
           dict(act=2), dict(x=72), dict(k=72), dict(ld=60), dict(hs=36)]
    if name == "attention":
        bad += [dict(heads=3), dict(heads=0), dict(window=-1), dict(first=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(y=72),
                dict(rows=1, seqs=1, width=1 << 26, ldt=1 << 26)]
        big = dict(rows=1, seqs=1, width=4096, ldt=4096)                       # long enough to be split, without the space
        assert S.lib().b2l_seq_paged_attention_work(1, 1, 4096, 16, 4, 2, 32, 32, 0, 0, 0, 0, 0, 0) > 0
        bad += [big, dict(big, work=64, floats=10), dict(work=72)]
    for kw in bad:
        rc = call(name, **dict(dict(rows=3), **kw))
        assert rc < 0 and S.lib().b2l_seq_last_error(), kw


# ----------------------------------------------------------------------------- units and splits, as csrc/seq_paged_attn.cuh counts them
def units_of(p_min, p_max, window, first, shift):
    size = 1 << shift
    end, lo = p_max + 1, max(p_min - window + 1, 0) if window else 0
    early = min(first if window else 0, lo)
    e = min((early + size - 1) >> shift, lo >> shift)
    n = 0 if end <= 0 else e + ((end + size - 1) >> shift) - (lo >> shift)
    return [(u if u < e else u - e + (lo >> shift)) << shift for u in range(n)]


@pytest.mark.parametrize("shift", [4, 5, 7])
def test_units_cover_what_is_seen_once_and_splits_cover_the_units(shift):
    size = 1 << shift
    for p_min, rows in ((-3, 2), (0, 1), (0, 5), (15, 1), (16, 1), (300, 40), (1000, 128), (517, 3)):
        for window, first in ((0, 0), (1, 0), (1, 1), (16, 16), (64, 4), (200, 130), (4096, 7), (90, 900)):
            p_max = p_min + rows - 1
            starts = units_of(p_min, p_max, window, first, shift)
            assert all(x % size == 0 and x >= 0 and x <= max(p_max, 0) for x in starts) and len(set(starts)) == len(starts)
            covered = {j for x in starts for j in range(x, x + size)}
            for p in range(max(p_min, 0), p_max + 1):
                assert all(j in covered for j in range(p + 1) if not window or j > p - window or j < first)
            for splits in (1, 2, 3, 7):
                per = -(-len(starts) // splits)
                got = [u for s in range(splits) for u in range(min(s * per, len(starts)), min(min(s * per, len(starts)) + per, len(starts)))]
                assert got == list(range(len(starts)))


def test_shares_of_row_tiles_cover_all_keys_once():
    """csrc/seq_paged_tc.cu: cuts at equal costs give every tile of keys of every row tile to one SM, the parts of a row tile to consecutive ones, and no SM
    more than one part that goes on and one that came from before."""
    source = open(os.path.join(os.path.dirname(paged.__file__), "csrc", "seq_paged_tc.cu")).read()
    extra, least, smallest = (int(x) for x in re.search(r"EXTRA = (\d+), LEAST = (\d+), SMALLEST_SHARE = (\d+);", source).groups())

    def cut(units, each, d):
        if d <= 0 or d >= extra + units * each:
            return 0 if d <= 0 else units
        y = max(d - extra, 0) // each
        return 0 if y < least else units if units - y < least else y

    rng = random.Random(1)
    for _ in range(300):
        tiles = [(max(rng.choice([0, 1, 2, 3, 4, 5, rng.randint(0, 40), rng.randint(0, 1000)]), 1), rng.choice([3, 4])) for _ in range(rng.choice([1, 2, 7, 60, 300]))]
        at = [0]
        for units, each in tiles:
            at.append(at[-1] + extra + units * each)
        ctas = rng.choice([1, 2, 5, 148])
        share = max(-(-at[-1] // ctas), smallest)
        parts, goes_on, came = [[] for _ in tiles], set(), set()
        for c in range(ctas):
            for i, (units, each) in enumerate(tiles):
                t0, t1 = (cut(units, each, min(x * share, at[-1]) - at[i]) for x in (c, c + 1))
                if t0 < t1:
                    parts[i].append((c, t0, t1))
                    if t1 - t0 < units:
                        side = goes_on if t0 == 0 else came
                        assert c not in side
                        side.add(c)
        for (units, _), mine in zip(tiles, parts):
            assert [t0 for _, t0, _ in mine] == [0] + [t1 for _, _, t1 in mine[:-1]] and mine[-1][2] == units
            assert [c for c, _, _ in mine] == list(range(mine[0][0], mine[0][0] + len(mine)))


def test_the_oracle_sees_what_the_formula_says():
    c = cache(dtype=torch.float32, kv_heads=1, dim=16, vdim=16)
    c.k.normal_()
    c.v.normal_()
    q = torch.randn(3, 2, 16)
    seqs = [(3, 20, [2, 1])]
    got, _, _ = O.attend(q, c, seqs, 0.3, window=4, first=2)
    for i, p in enumerate((17, 18, 19)):
        j = torch.tensor([x for x in range(p + 1) if x > p - 4 or x < 2])
        k, v = c.k[[2, 1]].transpose(1, 2).reshape(-1, 16)[j].double(), c.v[[2, 1]].transpose(1, 2).reshape(-1, 16)[j].double()
        for h in range(2):
            w = torch.exp(0.3 * k @ q[i, h].double())
            torch.testing.assert_close(got[i, h], (w[:, None] * v).sum(0) / w.sum(), rtol=1e-12, atol=1e-12)


@pytest.mark.parametrize("rows,heads", [(1, 4), (1, 1), (5, 1), (5, 4)])
def test_rows_as_the_kernels_take_them(rows, heads):
    """Whatever the strides: entries of a head consecutive, tokens and heads at multiples of 16 bytes, and the values are the same."""
    c, s = cache(), PagedStep.of([(rows, rows, [0])], CPU)
    wide = torch.randn(rows + 1, heads * 32 + 11).to(torch.bfloat16)
    flat = torch.randn(rows * heads * 33 + 1).to(torch.bfloat16)
    for x in (wide[:rows, :heads * 32].unflatten(1, (heads, 32)), wide[1:, 1:1 + heads * 32].unflatten(1, (heads, 32)), flat[1:1 + rows * heads * 32].view(rows, heads, 32),
              flat[:-1].view(rows, heads, 33)[..., :32], flat[:-1].view(rows, heads, 33)[..., 1:], flat[:rows * heads * 32].view(heads, rows, 32).transpose(0, 1),
              flat[:rows * heads * 32].view(rows, 32, heads).transpose(1, 2), flat[:32].expand(rows, heads, 32), flat[1:33].expand(rows, heads, 32)):
        y, s0, s1 = c._rows(x, heads, 32, s, "rows")
        assert s0 % 8 == 0 and s1 % 8 == 0 and y.data_ptr() % 16 == 0
        at = y.storage_offset()
        assert torch.equal(torch.as_strided(y, (rows, heads, 32), (s0, s1, 1), at), x)


@pytest.mark.parametrize("name", ["write", "read", "attention"])
def test_the_c_entries_have_nothing_to_do_without_rows_or_sequences(name):
    """Empty tensors have no address; sizes are looked at all the same."""
    none = dict(x=None, y=None, starts=None, lengths=None, table=None)
    assert call(name, **none) == 0 and call(name, rows=3, seqs=0, starts=None, lengths=None, table=None) == 0
    for kw in (dict(page=24), dict(K=24), dict(seqs=-1), dict(kv_heads=0), dict(act=2)):
        assert call(name, **dict(none, **kw)) < 0, kw


@pytest.mark.parametrize("seed", range(20))
def test_queries_are_multiplied_only_when_all_warps_have_them_there(seed):
    """csrc/seq_paged_tc.cu: eight softmax warps arrive at one barrier for every row tile.  One of them takes long over a row tile's outputs (rows computed again),
    others' waits may run out meanwhile: they go on without waiting, and what they do must not complete a row tile's phase before the slow one has come."""
    source = open(os.path.join(os.path.dirname(paged.__file__), "csrc", "seq_paged_tc.cu")).read()
    arrivals = re.findall(r"(if \(!dead\) )?mbar_arrive\(bar\(ct\.q_full\)\)", source)
    assert len(arrivals) == 1
    guarded, rng, warps, tiles = bool(arrivals[0]), random.Random(seed), 8, 4
    slow, slow_at = rng.randrange(warps), rng.randrange(tiles - 1)
    gave_up, came, phase, count = [False] * warps, [0] * warps, 0, 0          # came: row tiles whose queries the warp has put there
    released = False
    for _ in range(2000):
        w = rng.randrange(warps)
        if came[w] == tiles:
            continue
        if came[w] > phase and not gave_up[w]:                                 # waits for the products of its row tile
            if rng.random() < 0.1 and not released and came[slow] == slow_at + 1:
                gave_up[w] = w != slow
            continue
        if w == slow and came[w] == slow_at + 1 and not released:              # still at the outputs of the row tile before
            released = rng.random() < 0.02
            continue
        came[w] += 1
        if guarded and gave_up[w]:
            continue
        count += 1
        if count == warps:
            assert min(came) > phase, (came, phase)
            phase, count = phase + 1, 0


def test_windows_and_first_tokens_beyond_every_position_are_none():
    """A table of 4 pages of 16 has positions 0 .. 63: what is longer hides nothing, and what does not fit the C entry's int never reaches it."""
    c, s = cache(), PagedStep.of([(2, 2, [0])], CPU, width=4)
    whole = c._plan(2, 4, None, 0, 0, s)
    assert c._plan(2, 4, None, 63, 3, s)[1][8:10] == (63, 3) and whole[1][8:10] == (0, 0)
    for window, first in ((64, 0), (64, 3), (2 ** 31 - 1, 0), (2 ** 31, 7), (2 ** 32 + 5, 2 ** 40), (5, 64), (5, 2 ** 32 + 1)):
        assert c._plan(2, 4, None, window, first, s) == whole
