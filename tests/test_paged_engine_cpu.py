"""CPU: the engine's scheduler over a model that books pages, with a model that has no weights: its logits tell which tokens its sequence has had."""
import pytest
import torch

import lit_llama_b200 as P
from lit_llama_b200 import PagePool
from lit_llama_b200.state import PoolFull


class Told:
    """A model whose next token depends on every token of its sequence and its place, and whose calls number `fails` find no page."""
    graph_safe = False
    vocab, dtype, device = 97, torch.bfloat16, torch.device("cpu")

    def __init__(self, fails=()):
        self.seen, self.fails, self.calls = {}, set(fails), 0

    def state_specs(self):
        return {}

    def book(self, slot, pos0, n):
        pass

    def forward_portion(self, tokens, ctx, want=None):
        slot, pos0 = ctx.meta.tolist()
        self.calls += 1
        if self.calls in self.fails:
            raise PoolFull("no page")
        self.book(slot, pos0, tokens.numel())
        if pos0 == 0:
            self.seen[slot] = []
        assert len(self.seen[slot]) == pos0
        out = torch.zeros(tokens.numel(), self.vocab)
        for i, t in enumerate(tokens.tolist()):
            self.seen[slot].append(t)
            out[i, sum((j + 1) * x for j, x in enumerate(self.seen[slot])) % self.vocab] = 1.0
        return out if want is None else out[want.long()]


def serve(model, requests, n_slots=2, chunk=16, tries=1):
    engine = P.Engine(model, n_slots=n_slots, prefill_chunk=chunk)
    for rid, (prompt, n) in requests.items():
        engine.add_request(rid, prompt, n)
    for left in range(tries, 0, -1):
        try:
            return engine.run()
        except PoolFull:
            if left == 1:
                raise


def requests(*sizes):
    return {i: ([(7 * j + 3 * i) % 97 for j in range(length)], n) for i, (length, n) in enumerate(sizes)}


@pytest.mark.parametrize("fails", [[1], [2], [3], [4], [5], [6], [7], [2, 3], [1, 4, 9, 10], [5, 7, 9, 11, 13]])
def test_a_portion_that_could_not_run_is_run_again(fails):
    asked = requests((40, 5), (33, 7), (16, 3))
    assert serve(Told(fails), asked, tries=len(fails) + 1) == serve(Told(), asked)


class Paged(Told):
    """The same with pages that all slots share."""

    def __init__(self, n_pages, window=0, first=0):
        super().__init__()
        self.pages = PagePool(n_pages, 16, torch.device("cpu"), window=window, first=first)

    def release_slot(self, slot):
        if self.pages.has(slot):
            self.pages.release(slot)

    def has_room(self, live, tokens, portion):
        return self.pages.has_room(live, tokens, portion)

    def book(self, slot, pos0, n):
        if pos0 == 0:
            self.release_slot(slot)
        assert pos0 == 0 or self.pages.position(slot) == pos0
        self.pages.step([(slot, n)])


@pytest.mark.parametrize("n_pages,window,first,sizes", [
    (5, 0, 0, [(20, 40), (80, 1)]),                         # the second needs every page
    (5, 0, 0, [(1, 80), (80, 1), (5, 3)]),
    (6, 0, 0, [(16, 17), (17, 16), (40, 50), (90, 7), (1, 1)]),
    (12, 0, 0, [(60, 60), (60, 60), (3, 100), (100, 3)]),
    (6, 24, 2, [(23, 150), (70, 40), (5, 5)]),              # a window: pages for what it reaches
    (11, 24, 2, [(23, 150), (70, 40), (5, 5), (33, 60)]),
])
def test_requests_wait_for_pages(n_pages, window, first, sizes):
    """More slots than pages suffice for: everything is served, each request as it is alone, and all pages come back."""
    asked = requests(*sizes)
    model = Paged(n_pages, window, first)
    assert serve(model, asked, n_slots=4) == serve(Told(), asked)
    assert model.pages.free_pages() == n_pages


def test_a_request_that_is_larger_than_all_pages():
    """It runs by itself until the pages are used up and is then refused, as often as it is asked for; what was served before is not lost."""
    model = Paged(5)
    engine = P.Engine(model, n_slots=3, prefill_chunk=16)
    for rid, (prompt, n) in requests((20, 4), (30, 100)).items():
        engine.add_request(rid, prompt, n)
    for _ in range(2):
        with pytest.raises(PoolFull, match="pages"):
            engine.run()
    assert engine.finished[0].output == serve(Told(), requests((20, 4)))[0] and model.seen[0] and engine.live[1].fed == 30
    assert not engine.live[1].done and len(engine.live[1].output) == 5 * 16 - 30 + 1


@pytest.mark.parametrize("taken,enough", [(64, True), (80, False)])
def test_pages_that_another_user_of_the_pool_has_for_a_while(taken, enough):
    """A request that finds no page waits while others run; where nothing runs the shortage is reported, and nothing of any request is lost."""
    asked = requests((31, 20), (18, 14))                    # 4 and 2 pages: the first is at its third long before the second ends
    model = Paged(8)
    engine = P.Engine(model, n_slots=2, prefill_chunk=16)
    for rid, (prompt, n) in asked.items():
        engine.add_request(rid, prompt, n)
    engine._admit()
    model.pages.step([("elsewhere", taken)])                # booked after both were let in
    if not enough:
        with pytest.raises(PoolFull, match="pages"):
            engine.run()
        model.pages.release("elsewhere")
    assert engine.run() == serve(Told(), asked)


@pytest.mark.parametrize("window,first", [(0, 0), (1, 0), (16, 0), (17, 3), (40, 16), (33, 17), (100, 130)])
@pytest.mark.parametrize("portion", [1, 7, 16, 33])
def test_the_most_pages_of_a_sequence(window, first, portion):
    for total in (1, 15, 16, 17, 64, 100, 333):
        p = PagePool(64, 16, torch.device("cpu"), window=window, first=first)
        most, at = 0, 0
        while at < total:
            n = min(portion, total - at)
            p.step([("a", n)])
            at += n
            most = max(most, 64 - p.free_pages())
        assert most <= p.most_pages(total, portion) <= most + (1 + (first % 16 > 0) if window else 0)
        assert p.most_pages(total, portion) <= p.most_pages(total)


def test_room_beside_others():
    p = PagePool(8, 16, torch.device("cpu"))
    assert p.has_room({}, 128) and not p.has_room({}, 129)
    p.step([("a", 20), ("other", 1)])                       # a has 2 pages and will have 4; other has 1
    assert p.has_room({"a": 64}, 48) and not p.has_room({"a": 64}, 49)
    assert p.has_room({"a": 64, "new": 16}, 32) and not p.has_room({"a": 64, "new": 17}, 32)


def paged_llama(**kw):
    """A PagedLLaMAModel whose pages can be looked at without a device."""
    from types import SimpleNamespace as N

    config = N(padded_vocab_size=96, n_head=2, n_embd=32, n_layer=1, block_size=64)
    wte = torch.nn.Embedding(96, 32, dtype=torch.bfloat16)
    return P.PagedLLaMAModel(N(config=config, transformer=N(wte=wte), parameters=wte.parameters), **dict(dict(pages=8, page=16), **kw))


def test_engines_that_share_a_model_have_slots_of_their_own():
    model = paged_llama()
    a, b = P.Engine(model, n_slots=2), P.Engine(model, n_slots=2)
    for engine in (a, b):
        engine.pool.acquire("r")
        engine.model.book(0, 0, 20)                        # both in slot 0
    assert model.pages.free_pages() == 4
    assert not a.model.has_room({0: 64}, 48, 16) and a.model.has_room({0: 48}, 48, 16)      # the other engine's two pages are not free
    b.model.book(0, 20, 20)
    with pytest.raises(RuntimeError, match="position"):
        a.model.book(0, 40, 1)
    a.model.book(0, 20, 5)
    a.pool.release("r")
    assert model.pages.free_pages() == 5 and b.model.book(0, 40, 1).lengths.tolist() == [41]
    b.pool.release("r")
    assert model.pages.free_pages() == 8


def test_an_engine_that_goes_gives_its_pages_back():
    import gc

    model = paged_llama()
    a, b = P.Engine(model, n_slots=2), P.Engine(model, n_slots=2)
    a.pool.acquire("r")
    a.model.book(0, 0, 40)
    b.pool.acquire("r")
    b.model.book(0, 0, 20)
    model.book(0, 0, 5)                                    # a caller's own, without an engine
    assert model.pages.free_pages() == 2
    del a
    gc.collect()
    assert model.pages.free_pages() == 5
    del b
    gc.collect()
    assert model.pages.free_pages() == 7
    model.release_slot(0)
    assert model.pages.free_pages() == 8


def test_a_model_that_is_not_in_bf16_is_refused():
    """Its embedding's bytes would be read as bf16."""
    from types import SimpleNamespace as N

    model = paged_llama().model
    wte = torch.nn.Embedding(96, 32)
    with pytest.raises(RuntimeError, match="float32"):
        P.PagedLLaMAModel(N(config=model.config, transformer=N(wte=wte), parameters=wte.parameters), pages=8, page=16)


def test_a_portion_that_fails_after_its_pages_were_booked_can_be_run_again():
    for window in (0, 24):
        model = paged_llama(window=window)
        for slot, lengths in ((0, [5]), (1, [20, 16, 7, 16])):
            at = 0
            for n in lengths:
                model.book(slot, at, n)
                at += n
            free, pages = model.pages.free_pages(), model.pages.pages((model._owner, slot))
            with pytest.raises(MemoryError):
                with model.booked(slot, at, 30):
                    raise MemoryError
            kept = model.pages.pages((model._owner, slot))
            assert model.pages.position((model._owner, slot)) == at and model.pages.free_pages() >= free
            assert kept == [-1 if k < 0 else p for k, p in zip(kept, pages)]      # the same ones, but for those behind the window
            with model.booked(slot, at, 30) as step:
                assert step.lengths.tolist() == [at + 30]
            model.release_slot(slot)
        assert model.pages.free_pages() == 8


def test_a_step_that_could_not_be_made_books_nothing(monkeypatch):
    from lit_llama_b200 import PagedStep

    p = PagePool(8, 16, torch.device("cpu"))
    p.step([("a", 20)])
    before = p.pages("a")

    def none_left(*args, **kw):
        raise MemoryError
    with monkeypatch.context() as m:
        m.setattr(PagedStep, "of", none_left)
        with pytest.raises(MemoryError):
            p.step([("a", 30), ("b", 17), ("c", 0)])
    assert p.pages("a") == before and p.position("a") == 20 and p.requests() == ["a"] and p.free_pages() == 6
    assert p.step([("a", 30), ("b", 17)]).lengths.tolist() == [50, 17]


def test_tokens_that_did_not_come():
    p = PagePool(8, 16, torch.device("cpu"))
    p.step([("a", 20)])
    p.step([("a", 40)])
    with pytest.raises(ValueError):
        p.take_back("a", 61)
    p.take_back("a", 40)
    assert p.position("a") == 20 and p.free_pages() == 6
    p.take_back("a", 20)
    assert p.position("a") == 0 and p.pages("a") == [] and p.free_pages() == 8


def test_tokens_whose_window_is_gone_are_not_taken_back():
    """Pages that the window has left are other sequences' by now."""
    p = PagePool(12, 16, torch.device("cpu"), window=24, first=2)
    for n in (60, 40, 5):
        p.step([("a", n)])
    assert -1 in p.pages("a")
    free, pages = p.free_pages(), p.pages("a")
    with pytest.raises(ValueError, match="window"):
        p.take_back("a", 50)
    assert p.position("a") == 105 and p.free_pages() == free and p.pages("a") == pages
    p.take_back("a", 5)
    assert p.position("a") == 100
