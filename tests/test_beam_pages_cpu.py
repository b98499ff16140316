"""CPU: what a search copies and the pages that it needs while its beams become fewer."""
import math

import pytest
import torch

import lit_llama_b200 as P
import tree_oracle as T
from lit_llama_b200 import PagePool
from test_tree_cpu import CPU, Chain, selected  # noqa: F401


class Paged(Chain):
    """The same model with a page pool that is booked as the LLaMA with pages books it; `allowed(text)`: the tokens that may follow."""

    def __init__(self, allowed, pages, **kw):
        super().__init__(**kw)
        self.allowed, self.pages, self.copied, self.least = allowed, PagePool(pages, 16, CPU), [], pages

    def logits(self, text):
        x = super().logits(text)
        hidden = [t for t in range(self.vocab) if t not in self.allowed(list(text))]
        x[hidden] = -math.inf
        return x

    def release_slot(self, slot):
        super().release_slot(slot)
        if self.pages.has(slot):
            self.pages.release(slot)

    def forward_portion(self, tokens, ctx, want=None):
        self.pages.step([(ctx.meta.tolist()[0], tokens.numel())])
        return super().forward_portion(tokens, ctx, want)

    def reorder_slots(self, sources):
        self.copied.append(self.pages.reorder(sources))
        self.least = min(self.least, self.pages.free_pages())
        super().reorder_slots(sources)

    def forward_together(self, slots, positions, tokens):
        self.pages.step([(s, 1) for s in slots])
        return super().forward_together(slots, positions, tokens)


def search(model, beams, steps):
    engine = P.Engine(model, n_slots=beams)
    got = engine.beam_search([1, 2, 0], steps, beams)
    assert engine.pool.free_slots() == beams and model.pages.free_pages() == model.pages.n_pages and not model.seen
    return got


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("beams", [3, 4, 6])
@pytest.mark.parametrize("goes_on", [0, 1, 2])
def test_beams_that_become_fewer_take_no_page_more(goes_on, beams, seed, selected):  # noqa: F811
    """Every beam's tokens fill part of a page of its own, as many pages as beams.  Then only what came from one of the first tokens goes on, by two tokens; the others end."""
    def allowed(text):
        new = text[3:]
        if len(new) < 3:
            return range(6)
        return [t for t in (1, 4) if new[0] % 3 == goes_on] if len(new) == 3 else range(6)

    got = search(Paged(allowed, beams, vocab=6, seed=seed), beams, 6)
    assert got == search(Paged(allowed, 60, vocab=6, seed=seed), beams, 6)      # and with pages to spare


def test_what_goes_on_keeps_its_page(selected):  # noqa: F811
    """One of three beams goes on, whichever it is: nothing is copied for it."""
    for last in range(3):
        def allowed(text):
            new = text[3:]
            return range(3) if not new else [t for t in (2,) if new[0] == last] if len(new) == 1 else [0]

        model = Paged(allowed, 3, vocab=3, seed=5)
        assert [x for x, _ in search(model, 3, 4)] == [[last, 2, 0, 0]] and [len(c) for c in model.copied] == [2, 0, 0]


def test_the_oracle_selects_what_goes_on():
    x = torch.full((2, 4), -math.inf)
    x[1, 2] = 0.5
    assert [v.tolist() for v in T.select(x, torch.zeros(2), 1)] == [[0.0], [1], [2]]
