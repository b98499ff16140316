"""CPU: pages that sequences share, what the new entries refuse, and the engine's searches over models without weights."""
import ctypes as C
import itertools
import math
import random

import pytest
import torch

import lit_llama_b200 as P
import tree_oracle as T
from lit_llama_b200 import PagedCache, PagedLayers, PagedStep, PagedTree, PagePool, beam_select
from lit_llama_b200 import _seqlib as S
from lit_llama_b200.state import PagesFull, PoolFull

CPU = torch.device("cpu")


# ----------------------------------------------------------------------------- pages that sequences share
class Memory:
    """What lies in the pages of a pool: every booked token is written where the step's table says, copies are made as the pool asks for them."""

    def __init__(self, **kw):
        self.pool = PagePool(**dict(dict(n_pages=24, page=16, device=CPU), **kw))
        self.at, self.texts, self.next = {}, {}, 0

    def copy(self, pairs):
        assert len({b for _, b in pairs}) == len(pairs) and not {a for a, _ in pairs} & {b for _, b in pairs}
        for a, b in pairs:
            for place in range(16):
                if (a, place) in self.at:
                    self.at[b, place] = self.at[a, place]

    def step(self, entries):
        step = self.pool.step(entries)
        for b, (rid, n) in enumerate(entries):
            text = self.texts.setdefault(rid, [])
            for _ in range(n):
                self.next += 1
                text.append(self.next)
                p = len(text) - 1
                self.at[int(step.table[b, p // 16]), p % 16] = self.next

    def check(self):
        held = {}
        for rid, text in self.texts.items():
            pages = self.pool.pages(rid)
            assert self.pool.position(rid) == len(text) and len(pages) == -(-len(text) // 16)
            for p in pages:
                if p >= 0:
                    held[p] = held.get(p, 0) + 1
            reach = len(text) - self.pool.window + 1 if self.pool.window else 0
            for j, token in enumerate(text):
                if j >= reach or j < self.pool.first:
                    assert self.at[pages[j // 16], j % 16] == token, (rid, j)
        assert self.pool._shared == {p: n for p, n in held.items() if n > 1}
        assert sorted(self.pool._free + list(held)) == list(range(self.pool.n_pages))


@pytest.mark.parametrize("seed", range(12))
def test_forked_sequences_keep_their_tokens(seed):
    rng = random.Random(seed)
    m = Memory(**(dict(window=40, first=5) if seed % 3 == 2 else {}))
    for turn in range(250):
        ids = list(m.texts)
        what = rng.choice(["step", "step", "step", "fork", "reorder", "release", "take_back", "compact"])
        before = (dict(m.pool._length), {r: list(p) for r, p in m.pool._pages.items()}, list(m.pool._free), dict(m.pool._shared))
        try:
            if what == "step":
                some = rng.sample(ids + [f"n{turn}"], rng.randint(1, min(3, len(ids) + 1)))
                for rid in some:
                    if rid in m.texts:
                        m.copy(m.pool.own(rid))
                m.step([(rid, rng.choice([0, 1, 1, 3, 17])) for rid in some])
            elif what == "fork" and ids:
                s = rng.choice(ids)
                m.copy(m.pool.fork(s, f"f{turn}"))
                m.texts[f"f{turn}"] = list(m.texts[s])
            elif what == "reorder" and ids:
                after = rng.sample(ids, rng.randint(1, len(ids))) + [f"r{turn}"] * rng.randint(0, 1)
                sources = {rid: rng.choice(ids) for rid in after}
                m.copy(m.pool.reorder(sources))
                m.texts.update({r: list(text) for r, text in [(r, m.texts[s]) for r, s in sources.items()]})
            elif what == "release" and ids:
                rid = rng.choice(ids)
                m.pool.release(rid)
                del m.texts[rid]
            elif what == "take_back" and ids:
                rid = rng.choice(ids)
                n = rng.randint(0, min(len(m.texts[rid]), 20))
                m.pool.take_back(rid, n)
                del m.texts[rid][len(m.texts[rid]) - n:]
            elif what == "compact":
                m.copy(m.pool.compact())
                used = {p for r in m.texts for p in m.pool.pages(r) if p >= 0}
                assert used == set(range(len(used)))
        except PagesFull:
            if what in ("fork", "reorder"):
                assert before == (m.pool._length, m.pool._pages, m.pool._free, m.pool._shared)
            m.texts = {r: t for r, t in m.texts.items() if m.pool.has(r)}
            for rid in rng.sample(list(m.texts), len(m.texts) // 2):
                m.pool.release(rid)
                del m.texts[rid]
        except ValueError as e:                              # pages that the window had given back
            assert what == "take_back" and "given back" in str(e)
        m.check()


def test_only_what_goes_on_being_written_is_copied():
    p = PagePool(8, 16, CPU)
    p.step([("a", 40)])
    assert p.pages("a") == [0, 1, 2]
    assert p.fork("a", "b") == [(2, 3)] and p.pages("b") == [0, 1, 3] and p.free_pages() == 4
    p.step([("a", 8), ("b", 8)])                             # up to the border: nothing to copy then
    assert p.fork("a", "c") == [] and p.pages("c") == [0, 1, 2]
    assert p.reorder({"a": "b", "b": "b"}) == [] and p.pages("a") == p.pages("b") == [0, 1, 3] and p.pages("c") == [0, 1, 2]
    p.step([("a", 1)])
    assert p.pages("a") == [0, 1, 3, 4]
    assert p.reorder({"a": "c", "b": "a"}) == []             # b goes on with a's last page, which nobody else has
    assert p.pages("b") == [0, 1, 3, 4] and p.pages("a") == [0, 1, 2]
    for rid in "abc":
        p.release(rid)
    assert p.free_pages() == 8 and not p._shared


def test_room_counts_the_copy_of_a_page_that_others_have_too():
    p = PagePool(4, 16, CPU)
    p.step([("a", 32)])
    p.fork("a", "b")
    p.take_back("b", 5)                                      # goes on in a page that a keeps
    assert p.has_room({"b": 32}, 16) and not p.has_room({"b": 32}, 17)
    p.own("b")
    assert p.has_room({"b": 32}, 16) and not p.has_room({"b": 32}, 17)
    p.step([("b", 5), ("new", 16)])
    assert p.free_pages() == 0


def test_a_shared_page_is_not_written():
    p = PagePool(8, 16, CPU)
    p.step([("a", 32)])
    assert p.fork("a", "b") == []
    p.take_back("b", 5)                                      # into a page that both have
    with pytest.raises(ValueError, match="own first"):
        p.step([("b", 1)])
    assert p.position("b") == 27
    p.step([("b", 0)])
    assert p.own("a") == [] and p.own("b") == [(1, 2)] and p.own("b") == []
    assert p.step([("b", 1)]).table.tolist() == [[0, 2]]
    with pytest.raises(ValueError, match="already"):
        p.fork("a", "b")
    with pytest.raises(KeyError):
        p.reorder({"a": "x"})
    full = PagePool(2, 16, CPU)
    full.step([("a", 17)])
    with pytest.raises(PagesFull):
        full.fork("a", "b")
    assert not full.has("b") and full.pages("a") == [0, 1]
    full.take_back("a", 1)
    full.fork("a", "b")
    full.take_back("b", 1)
    full.step([("a", 1)])
    with pytest.raises(PagesFull):
        full.own("b")


def test_room_beside_sequences_that_share_pages():
    p = PagePool(8, 16, CPU)
    p.step([("a", 64)])
    p.fork("a", "b")
    assert p.has_room({"a": 64}, 64) and not p.has_room({"a": 64, "b": 64}, 16)      # what both have is there once, and may have to be there twice


def test_windows_give_shared_pages_back_when_the_last_one_moves_on():
    p = PagePool(6, 16, CPU, window=16)
    p.step([("a", 32)])
    p.fork("a", "b")
    p.step([("a", 16)])
    assert p.pages("a")[0] == -1 and p.pages("b")[0] == 0 and p.free_pages() == 3
    p.step([("b", 16)])
    assert p.free_pages() == 3 and p.pages("b")[0] == -1


# ----------------------------------------------------------------------------- refusals
def cache(**kw):
    return PagedCache.empty(**dict(dict(n_pages=4, page=16, kv_heads=2, dim=32, vdim=16, device="cpu"), **kw))


def test_the_kernels_run_on_cuda_only():
    c, s = cache(), PagedStep.of([(2, 2, [0])], CPU)
    ints = torch.zeros(2, dtype=torch.int32)
    for call in (lambda: PagedTree(s, ints), lambda: PagedLayers([c]).copy([(0, 1)]), lambda: PagedLayers([c]).keep(s, ints, ints), lambda: beam_select(torch.zeros(1, 2, 9), torch.zeros(1, 2), 3)):
        with pytest.raises(RuntimeError, match="CUDA only"):
            call()
    PagedLayers([c]).copy([])


def test_calls_that_do_not_fit_are_refused():
    s = PagedStep.of([(2, 2, [0])], CPU)
    ints = torch.zeros(2, dtype=torch.int32)
    for parents in (ints.long(), ints[:1], ints[None], torch.zeros(4, dtype=torch.int32)[::2]):
        with pytest.raises(ValueError):
            PagedTree(s, parents)
    for kw in (dict(nodes=-1), dict(window=-1), dict(first=-1)):
        with pytest.raises(ValueError):
            PagedTree(s, ints, **kw)
    with pytest.raises(ValueError):
        PagedLayers([])
    for other in (cache(n_pages=5), cache(dim=48), cache(store="int8"), cache(dtype=torch.float32)):
        with pytest.raises(ValueError, match="different"):
            PagedLayers([cache(), other])
    layers = PagedLayers([cache(), cache()])
    for pairs in ([(0, 4)], [(-1, 2)], [(0, 1), (2, 1)], [(0, 1), (1, 2)], torch.zeros(3, dtype=torch.int32), torch.zeros(2, 2)):
        with pytest.raises(ValueError):
            layers.copy(pairs)
    for kept, counts in ((ints.long(), ints[:1]), (ints[:1], ints[:1]), (ints, ints[:0])):
        with pytest.raises(ValueError):
            layers.keep(s, kept, counts)
    x, sc = torch.zeros(1, 2, 9), torch.zeros(1, 2)
    for bad in (dict(logits=x[0]), dict(logits=x.half()), dict(scores=sc[0]), dict(scores=sc.double()), dict(count=0), dict(count=19), dict(logits=torch.zeros(1, 65, 9), scores=torch.zeros(1, 65))):
        with pytest.raises(ValueError):
            beam_select(**dict(dict(logits=x, scores=sc, count=3), **bad))


def test_the_c_entries_refuse_before_they_launch():
    """Pointers that are never followed: every call is refused, or has nothing to do."""
    lib = S.lib()
    pools = (C.c_void_p * 4)(64, 64, None, None)
    eight = (C.c_void_p * 4)(64, 64, 64, 64)
    at = C.addressof(pools)

    def build(parents=64, starts=64, lengths=64, masks=64, words=1, depths=64, positions=64, rows=3, seqs=0, window=0, first=0):
        return lib.b2l_seq_tree_build(parents, starts, lengths, masks, words, depths, positions, rows, seqs, window, first, None)

    def accept(logits=64, ld=9, noise=None, ldn=9, temperature=0.0, parents=64, starts=64, tokens=64, wide=0, kept=64, counts=64, next_=64, work=64, size=1 << 20, rows=3, seqs=0, vocab=9, act=1):
        return lib.b2l_seq_tree_accept(logits, ld, noise, ldn, temperature, parents, starts, tokens, wide, kept, counts, next_, work, size, rows, seqs, vocab, act, None)

    def keep(pools=at, layers=1, starts=64, lengths=64, table=64, ldt=4, width=4, kept=64, counts=64, rows=3, seqs=0, pages=4, page=16, kv=2, K=32, V=32, store=0, act=0):
        return lib.b2l_seq_paged_keep(pools, layers, starts, lengths, table, ldt, width, kept, counts, rows, seqs, pages, page, kv, K, V, store, act, None)

    def copy(pools=at, layers=1, pairs=64, n=0, pages=4, page=16, kv=2, K=32, V=32, store=0, act=0):
        return lib.b2l_seq_paged_copy(pools, layers, pairs, n, pages, page, kv, K, V, store, act, None)

    def select(logits=64, ld=9, scores=64, values=64, of=64, tokens=64, work=64, size=1 << 20, groups=0, beams=2, vocab=9, count=4, act=1):
        return lib.b2l_seq_beam_select(logits, ld, scores, values, of, tokens, work, size, groups, beams, vocab, count, act, None)

    def attend(q=64, ld=64, hs=32, k=64, masks=64, words=1, depths=64, out=64, work=None, floats=0, rows=3, seqs=0, heads=4, kv=2, K=32, window=0, scale=1.0, width=4, act=0, store=0):
        return lib.b2l_seq_paged_attention_tree(q, ld, hs, k, 64, None, None, 64, 64, 64, width, width, masks, words, depths, 1, out, work, floats, rows, seqs, 4, 16, heads, kv, K, 32, window, 0,
                                                scale, 0, 0, store, act, None)

    bad = {build: [dict(parents=None), dict(masks=None), dict(words=0), dict(rows=-1), dict(seqs=-1), dict(window=-1), dict(first=-1), dict(depths=None), dict(positions=None), dict(rows=1 << 30)],
           accept: [dict(logits=None), dict(ld=8), dict(parents=None), dict(starts=None), dict(tokens=None), dict(kept=None), dict(counts=None), dict(next_=None), dict(work=None), dict(size=10),
                    dict(work=72), dict(rows=-1), dict(vocab=0), dict(rows=65536), dict(noise=64, temperature=0.0), dict(noise=64, temperature=1.0, ldn=8),
                    dict(noise=64, temperature=float("nan")), dict(act=2)],
           keep: [dict(pools=None), dict(layers=-1), dict(starts=None), dict(lengths=None), dict(table=None), dict(kept=None), dict(counts=None), dict(page=24), dict(K=24), dict(store=1), dict(act=2),
                  dict(ldt=3), dict(seqs=65536), dict(pages=1 << 27)],
           copy: [dict(pools=None), dict(layers=-1), dict(pairs=None), dict(pairs=68), dict(n=-1), dict(n=65536), dict(page=8), dict(V=8), dict(store=3), dict(kv=0), dict(store=2)],
           select: [dict(logits=None), dict(ld=8), dict(scores=None), dict(values=None), dict(of=None), dict(tokens=None), dict(work=None), dict(size=5), dict(work=72), dict(beams=0), dict(beams=65),
                    dict(count=0), dict(count=19), dict(count=65, vocab=99, ld=99), dict(vocab=0), dict(groups=-1), dict(groups=40000), dict(act=2)],
           attend: [dict(q=None), dict(k=None), dict(masks=None), dict(words=0), dict(depths=None), dict(out=None), dict(q=72), dict(ld=60), dict(heads=3), dict(K=24), dict(window=-1),
                    dict(scale=0.0), dict(width=4096), dict(width=4096, work=64, floats=10), dict(act=2), dict(store=1)]}
    some = {build: dict(seqs=1), accept: dict(seqs=1), keep: dict(seqs=1), copy: dict(n=2), select: dict(groups=1), attend: dict(seqs=1)}
    for f, cases in bad.items():
        assert f() == 0, f
        for kw in cases:
            assert f(**dict(some[f], **kw)) < 0 and lib.b2l_seq_last_error(), (f.__name__, kw)
    assert keep(pools=C.addressof(eight), store=2, seqs=0) == 0 and copy(layers=0, n=2, pools=None) == 0
    assert lib.b2l_seq_tree_accept_work(0, 9) == 0 and lib.b2l_seq_beam_work(0, 2, 9, 4, 0) == 0
    assert lib.b2l_seq_tree_accept_work(3, 32000) >= 3 * 20 and lib.b2l_seq_beam_work(2, 2, 32000, 8, 1) >= 4 * (8 * 8 + 12)


# ----------------------------------------------------------------------------- the engine's searches
class Chain:
    """A model whose logits depend on all of a sequence's tokens, with slots that can be forked and trees; no weights, no pages."""
    graph_safe = False
    dtype, device = torch.bfloat16, CPU

    def __init__(self, vocab=5, seed=0, max_positions=0):
        self.vocab, self.seed, self.max_positions, self.seen, self.calls = vocab, seed, max_positions, {}, []

    def logits(self, text):
        g = torch.Generator().manual_seed(hash((self.seed,) + tuple(text)) % (2 ** 31))
        return torch.randn(self.vocab, generator=g) * 2

    def state_specs(self):
        return {}

    def release_slot(self, slot):
        self.seen.pop(slot, None)

    def forward_portion(self, tokens, ctx, want=None):
        slot, pos0 = ctx.meta.tolist()
        text = self.seen.setdefault(slot, [])
        assert len(text) == pos0
        out = []
        for t in tokens.tolist():
            text.append(t)
            out.append(self.logits(text))
        out = torch.stack(out)
        return out if want is None else out[want.long()]

    def reorder_slots(self, sources):
        self.seen.update([(s, list(text)) for s, text in [(s, self.seen[t]) for s, t in sources.items()]])

    def forward_together(self, slots, positions, tokens):
        self.calls.append(len(slots))
        for s, p, t in zip(slots, positions, tokens.tolist()):
            assert len(self.seen[s]) == p
            self.seen[s].append(t)
        return torch.stack([self.logits(self.seen[s]) for s in slots])

    def forward_tree(self, slot, pos0, tokens, parents):
        self.calls.append(tokens.numel())
        text, parents, tokens = self.seen[slot], parents.tolist(), tokens.tolist()
        assert len(text) == pos0 and all(-1 <= p < i for i, p in enumerate(parents))
        paths = []
        for i, p in enumerate(parents):
            paths.append((paths[p] if p >= 0 else []) + [tokens[i]])
        logits = torch.stack([self.logits(text + path) for path in paths])

        class Tree:
            def accept(self, logits, tokens, temperature=0.0):
                kept, last = T.accept(T.targets(logits), tokens.tolist(), parents)
                pad = torch.full((len(parents) - len(kept),), -1, dtype=torch.int32)
                return torch.cat([torch.tensor(kept, dtype=torch.int32), pad]), torch.tensor([len(kept)], dtype=torch.int32), torch.tensor([last], dtype=torch.int32)

        self.text = tokens
        return logits, Tree()

    def keep(self, slot, tree, kept, counts, n):
        self.seen[slot] += [self.text[i] for i in kept.tolist()[:n]]


@pytest.fixture
def selected(monkeypatch):
    def select(logits, scores, count):
        out = [T.select(x, s, count) for x, s in zip(logits, scores)]
        return torch.stack([v for v, _, _ in out]).float(), torch.stack([b for _, b, _ in out]).int(), torch.stack([t for _, _, t in out]).int()

    monkeypatch.setattr("lit_llama_b200.search.beam_select", select)


def total(model, prompt, new):
    return sum(float(torch.log_softmax(model.logits(prompt + new[:i]).double(), -1)[t]) for i, t in enumerate(new))


@pytest.mark.parametrize("seed", range(4))
def test_a_search_with_room_for_all_finds_the_best(seed, selected):
    prompt = [1, 2, 0, 3]
    engine = P.Engine(Chain(3, seed), n_slots=32, prefill_chunk=3)
    got = engine.beam_search(prompt, 4, 27)
    want = sorted(((total(engine.model, prompt, list(x)) / 4, list(x)) for x in itertools.product(range(3), repeat=4)), reverse=True)
    assert [x for x, _ in got] == [x for _, x in want[:27]] and engine.pool.free_slots() == 32 and not engine.model.seen
    assert all(math.isclose(s, w, rel_tol=1e-5, abs_tol=1e-5) for (_, s), (w, _) in zip(got, want))


@pytest.mark.parametrize("beams,eos,penalty", [(1, None, 1.0), (3, None, 1.0), (4, 2, 1.0), (4, 2, 0.0), (2, 0, 2.0)])
def test_beams_step_by_step(beams, eos, penalty, selected):
    """Against the same search written on lists of tokens."""
    prompt, steps = [3, 1], 6
    for seed in range(6):
        model = Chain(7, seed)
        live, done = [([], 0.0)], []
        for n in range(1, steps + 1):
            found = sorted(((s + float(lp), -w, -t) for w, (x, s) in enumerate(live) for t, lp in enumerate(torch.log_softmax(model.logits(prompt + x).double(), -1))), reverse=True)[:2 * beams]
            after = []
            for rank, (s, w, t) in enumerate(found):
                x = live[-w][0] + [-t]
                if -t == eos:
                    done += [(x, s / n ** penalty)] * (rank < beams)
                elif len(after) < beams:
                    after.append((x, s))
            done = sorted(done, key=lambda x: -x[1])[:beams]
            live = after
            if n == steps or (len(done) == beams and after[0][1] / n ** penalty <= done[-1][1]):
                done = sorted(done + [(x, s / n ** penalty) for x, s in after], key=lambda x: -x[1])[:beams]
                break
        engine = P.Engine(model, n_slots=beams)
        got = engine.beam_search(prompt, steps, beams, eos_id=eos, length_penalty=penalty)
        assert [x for x, _ in got] == [x for x, _ in done]
        assert all(math.isclose(a, b, rel_tol=1e-5) for (_, a), (_, b) in zip(got, done))
        assert engine.pool.free_slots() == beams and not model.seen


def test_searches_that_do_not_fit(selected):
    engine = P.Engine(Chain(), n_slots=3)
    for beams, n in ((0, 5), (33, 5), (2, 0)):
        with pytest.raises(ValueError):
            engine.beam_search([1], n, beams)
    with pytest.raises(ValueError, match="empty"):
        engine.beam_search([], 3, 2)
    with pytest.raises(PoolFull):
        engine.beam_search([1], 3, 4)
    with pytest.raises(PoolFull):
        P.Engine(Chain(max_positions=4), n_slots=3).beam_search([1, 2], 5, 2)
    small = P.Engine(Chain(), n_slots=3, max_tokens=9)
    with pytest.raises(PoolFull):
        small.beam_search([1, 2, 3], 5, 3)
    assert small.pool.free_slots() == 3 and engine.pool.free_slots() == 3 and not small.model.seen

    class Plain:
        graph_safe, vocab, dtype, device = False, 5, torch.bfloat16, CPU

        def state_specs(self):
            return {}

    for call in (lambda e: e.beam_search([1], 2, 1), lambda e: e.generate_drafted([1], 2, lambda t: ([], []))):
        with pytest.raises(RuntimeError, match="Plain"):
            call(P.Engine(Plain()))


@pytest.mark.parametrize("seed", range(5))
@pytest.mark.parametrize("kind", ["none", "right", "wrong", "trees"])
def test_drafts_change_the_steps_and_not_the_tokens(kind, seed):
    rng = random.Random(seed)
    prompt = [4, 0, 1, 1, 2]
    plain = P.Engine(Chain(5, seed), n_slots=1, prefill_chunk=2)
    want = plain.generate(prompt, 20)
    model = Chain(5, seed)

    def draft(text):
        assert text == want[:len(text)]
        if kind == "none":
            return [], []
        if kind == "right":
            return want[len(text):len(text) + 4], [-1, 0, 1, 2][:len(want) - len(text)]
        if kind == "wrong":
            return [(want[len(text)] + 1) % 5] * 3, [-1, -1, 0]
        n = rng.randint(0, 9)
        return [rng.randrange(5) for _ in range(n)], [rng.randint(-1, i - 1) for i in range(n)]

    engine = P.Engine(model, n_slots=1, prefill_chunk=2)
    assert engine.generate_drafted(prompt, 20, draft) == want and not model.seen and engine.pool.free_slots() == 1
    assert len(model.calls) == {"none": 19, "wrong": 19, "right": 4}.get(kind, len(model.calls))
    if kind == "trees":
        assert len(model.calls) < 19
    assert engine.generate_drafted(prompt, 0, draft) == prompt and engine.generate_drafted(prompt, 1, draft) == want[:6]
    eos = want[9]
    stop = want.index(eos, 5)
    assert engine.generate_drafted(prompt, 20, draft, eos_id=eos) == want[:stop + 1]


def test_drafts_that_do_not_fit():
    engine = P.Engine(Chain(max_positions=12), n_slots=1)
    for bad in (([1], []), ([1, 2], [-1, 1]), ([1], [-2])):
        with pytest.raises(ValueError, match="draft"):
            engine.generate_drafted([1, 2], 5, lambda t: bad)
    with pytest.raises(ValueError, match="empty"):
        engine.generate_drafted([], 5, lambda t: ([], []))
    with pytest.raises(PoolFull):                            # the thirteenth position
        engine.generate_drafted([1, 2, 3], 12, lambda t: ([0] * 30, [-1] * 30))
    assert len(engine.generate_drafted([1, 2, 3], 10, lambda t: ([0] * 30, [-1] * 30))) == 13
    assert engine.pool.free_slots() == 1 and not engine.model.seen
    small = P.Engine(Chain(), n_slots=1, max_tokens=8)
    assert len(small.generate_drafted([1, 2, 3], 6, lambda t: ([0] * 30, [-1] * 30))) == 9
    with pytest.raises(PoolFull):
        small.generate_drafted([1, 2, 3], 7, lambda t: ([0] * 30, [-1] * 30))
