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
