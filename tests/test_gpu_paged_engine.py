"""GPU: the LLaMA with its pages behind engines that share them: requests that wait for pages."""
import pytest

import lit_llama_b200 as P
from test_gpu_paged_llama import PROMPT, llama

pytestmark = pytest.mark.gpu

PROMPTS = {"a": PROMPT, "b": PROMPT[5:9], "c": PROMPT[::-1] + PROMPT[:3]}


def alone(model, n, **kw):
    out = {}
    for r, p in PROMPTS.items():
        engine = P.Engine(P.PagedLLaMAModel(model, pages=12, page=16, **kw), n_slots=1, prefill_chunk=9)
        engine.add_request(r, p, n)
        out.update(engine.run())
    return out


@pytest.mark.parametrize("kw,pages", [({}, 3), ({}, 5), (dict(window=20, first=2), 4)])
def test_requests_wait_for_pages(kw, pages):
    """As many slots as requests, pages for one or two of them."""
    model = llama()
    paged = P.PagedLLaMAModel(model, pages=pages, page=16, **kw)
    engine = P.Engine(paged, n_slots=3, prefill_chunk=9)
    for r, p in PROMPTS.items():
        engine.add_request(r, p, 20)
    assert engine.run() == alone(model, 20, **kw)
    assert paged.pages.free_pages() == pages
