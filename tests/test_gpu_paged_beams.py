"""GPU: the LLaMA with pages goes on from one prompt in several ways: trees of drafted tokens, sequences that share pages, beams."""
import random

import pytest
import torch

from test_gpu_paged_llama import BOUND, PROMPT, llama, rel

pytestmark = pytest.mark.gpu

DEV = "cuda"


def paged(store="act", **kw):
    import lit_llama_b200 as P

    return P.PagedLLaMAModel(llama(), **dict(dict(pages=16, page=16, store=store), **kw))


def whole(model, texts):
    """Logits of every token of each text, in one portion each, from an engine of its own."""
    import lit_llama_b200 as P

    engine, out = P.Engine(model, n_slots=1), []
    for i, text in enumerate(texts):
        out.append(engine.step([dict(id=i, tokens=list(text), want=list(range(len(text))))], end=[i])[0])
    return out


@pytest.mark.parametrize("store", ["act", "int8", "fp8"])
@pytest.mark.parametrize("window,first", [(0, 0), (24, 2)])
def test_a_tree_gives_each_token_what_its_path_alone_gives(window, first, store):
    """Two kernels for the same sums (a step of a tree and a portion): within the bound of the portions against each other."""
    model = paged(store, window=window, first=first)
    rng = random.Random(7)
    nodes = [rng.randrange(96) for _ in range(12)]
    parents = [-1] + [rng.randint(max(0, i - 4), i - 1) for i in range(1, 12)]
    paths = []
    for i, p in enumerate(parents):
        paths.append((paths[p] if p >= 0 else []) + [i])
    import lit_llama_b200 as P

    engine = P.Engine(model, n_slots=2)
    engine.step([dict(id="t", tokens=PROMPT)])
    m, slot = engine.model, engine.pool.slot("t")
    logits, tree = m.forward_tree(slot, len(PROMPT), torch.tensor(nodes, device=DEV), torch.tensor(parents, dtype=torch.int32, device=DEV))
    want = torch.stack([x[-1] for x in whole(model, [PROMPT + [nodes[j] for j in path] for path in paths])])
    assert rel(logits.float(), want) < BOUND[store]
    # the longest path is kept: what follows is what a sequence with its tokens gives
    path = max(paths, key=len)
    kept = torch.tensor(path + [-1] * (12 - len(path)), dtype=torch.int32, device=DEV)
    m.keep(slot, tree, kept, torch.tensor([len(path)], dtype=torch.int32, device=DEV), len(path))
    engine.pool.advance("t", len(path))
    assert m.pages.position((m._owner, slot)) == len(PROMPT) + len(path)
    got = engine.step([dict(id="t", tokens=[11, 12, 13], want=[0, 1, 2])])[0]
    assert rel(got, whole(model, [PROMPT + [nodes[j] for j in path] + [11, 12, 13]])[0][-3:]) < BOUND[store]


def test_sequences_that_are_forked_go_on_by_themselves():
    import lit_llama_b200 as P

    model = paged()
    engine = P.Engine(model, n_slots=3)
    ids = [("f", 0)]
    engine.step([dict(id=ids[0], tokens=PROMPT)])
    m = engine.model
    engine._reorder(ids, [0, 0, 0])
    assert len(ids) == 3 and m.pages.free_pages() == 16 - 2 - 2                 # one full page that they share, and the one that each goes on writing
    more = [[5, 6, 7], [50, 6, 70], [80, 81, 82]]
    for n in range(3):
        got = engine._together(ids, [x[n] for x in more])
        want = torch.stack([x[-1] for x in whole(model, [PROMPT + x[:n + 1] for x in more])])
        assert rel(got, want) < BOUND["act"]
    engine._reorder(ids, [2, 0])                                               # the second gives way
    assert len(ids) == 2
    got = engine._together(ids, [1, 2])
    want = torch.stack([x[-1] for x in whole(model, [PROMPT + more[2] + [1], PROMPT + more[0] + [2]])])
    assert rel(got, want) < BOUND["act"]
    for rid in ids:
        engine.pool.release(rid)
    assert m.pages.free_pages() == 16


@pytest.mark.parametrize("store", ["act", "int8"])
def test_beams_of_the_model(store):
    """Every continuation's sum of log-probabilities is what one portion over it gives: a logit is off by BOUND of the logits' norm over the vocabulary at most, the
    log-probability of a token by twice that."""
    import lit_llama_b200 as P

    model = paged(store)
    engine = P.Engine(model, n_slots=5, prefill_chunk=8)
    got = engine.beam_search(PROMPT, 12, 4, length_penalty=0.0)
    assert len(got) == 4 and len({tuple(x) for x, _ in got}) == 4 and model.pages.free_pages() == 16 and engine.pool.free_slots() == 5
    for (x, score), logits in zip(got, whole(model, [PROMPT + x for x, _ in got])):
        lp = torch.log_softmax(logits.double(), -1)
        mine = sum(float(lp[len(PROMPT) - 1 + i, t]) for i, t in enumerate(x))
        assert abs(mine - score) < 12 * 2 * BOUND[store] * float(logits.norm(dim=-1).max())
    assert [s for _, s in got] == sorted((s for _, s in got), reverse=True)
    assert engine.beam_search(PROMPT, 12, 4, length_penalty=0.0) == got
    one = engine.beam_search(PROMPT, 6, 1)[0][0]
    eos = one[2]
    cut = engine.beam_search(PROMPT, 6, 1, eos_id=eos)
    assert cut[0][0] == one[:one.index(eos) + 1]


@pytest.mark.parametrize("store", ["act", "fp8"])
def test_drafted_tokens_are_the_models_own(store):
    """Greedy: every token's logit is within the bound of the largest of one portion over the result; good guesses take fewer steps."""
    import lit_llama_b200 as P

    model = paged(store)
    engine = P.Engine(model, n_slots=2, prefill_chunk=8)
    plain = engine.generate(PROMPT, 24)
    rng = random.Random(3)

    def right(text):
        return plain[len(text):len(text) + 5], [-1, 0, 1, 2, 3][:max(len(plain) - len(text), 0)]

    def some(text):                                                            # a tree with the right tokens somewhere in it
        out, parents, last = [], [], -1
        for t in plain[len(text):len(text) + 3]:
            for _ in range(rng.randint(0, 2)):
                out.append(rng.randrange(96))
                parents.append(last)
            out.append(t)
            parents.append(last)
            last = len(out) - 1
        return out, parents

    for draft in (right, some, lambda text: ([1, 2], [-1, -1]), lambda text: ([], [])):
        before = engine.steps
        got = engine.generate_drafted(PROMPT, 24, draft)
        assert len(got) == len(PROMPT) + 24 and got[:len(PROMPT)] == PROMPT
        logits = whole(model, [got])[0]
        for i in range(len(PROMPT), len(got)):
            row = logits[i - 1]
            assert float(row.max() - row[got[i]]) <= 2 * BOUND[store] * float(row.norm())
        if got == plain and draft in (right, some):
            assert engine.steps - before < 3 + 24 / 2
    assert model.pages.free_pages() == 16 and engine.pool.free_slots() == 2
    drawn = engine.generate_drafted(PROMPT, 16, some, temperature=1.5)
    assert len(drawn) == len(PROMPT) + 16 and all(0 <= t < model.vocab for t in drawn)      # (the padded vocabulary)


def test_drafts_without_pages_left():
    """A pool that just holds the sequence: guesses that do not fit are left out."""
    import lit_llama_b200 as P

    model = paged(pages=3)
    engine = P.Engine(model, n_slots=1)
    plain = engine.generate(PROMPT, 20)
    got = engine.generate_drafted(PROMPT, 20, lambda text: ([0] * 40, [-1] * 40))
    assert len(got) == len(plain) and model.pages.free_pages() == 3


def test_beams_that_find_no_page():
    import lit_llama_b200 as P
    from lit_llama_b200.state import PagesFull

    model = paged(pages=4)
    engine = P.Engine(model, n_slots=8)
    with pytest.raises(PagesFull):
        engine.beam_search(PROMPT, 30, 8)
    assert model.pages.free_pages() == 4 and engine.pool.free_slots() == 8
    assert len(engine.beam_search(PROMPT, 8, 2)) == 2
