"""GPU: the LLaMA with its pages behind engines that share them: requests that wait for pages, engines side by side."""
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


def test_two_engines_side_by_side():
    """Both have their request in slot 0, at the same positions, and take turns."""
    import torch

    model = llama()
    prompts = [PROMPT, PROMPT[::-1]]
    want = []
    for p in prompts:
        engine = P.Engine(P.PagedLLaMAModel(model, pages=12, page=16), n_slots=1)
        want.append(torch.cat([engine.step([dict(id=0, tokens=part, want=list(range(len(part))))])[0] for part in (p[:9], p[9:17], p[17:18], p[18:])]))
    paged = P.PagedLLaMAModel(model, pages=12, page=16)
    engines, got = [P.Engine(paged, n_slots=1) for _ in prompts], [[], []]
    for i, j in ((0, 9), (9, 17), (17, 18), (18, 23)):
        for engine, p, out in zip(engines, prompts, got):
            out += engine.step([dict(id=0, tokens=p[i:j], want=list(range(j - i)))])
    for a, b in zip(got, want):
        assert torch.equal(torch.cat(a), b)
    assert paged.pages.free_pages() == 8
    del engine, engines
    assert paged.pages.free_pages() == 12


def test_a_portion_that_fails_midway_can_be_run_again():
    import torch

    model = llama()
    want = P.Engine(P.PagedLLaMAModel(model, pages=12, page=16), n_slots=1).step([dict(id=0, tokens=PROMPT, want=[22])])[0]
    paged = P.PagedLLaMAModel(model, pages=12, page=16)
    engine = P.Engine(paged, n_slots=1)
    engine.step([dict(id=0, tokens=PROMPT[:9])])
    last, attend = paged.caches[-1], paged.caches[-1].attend

    def no_memory(*args, **kw):
        raise torch.cuda.OutOfMemoryError("none left")
    last.attend = no_memory
    with pytest.raises(torch.cuda.OutOfMemoryError):
        engine.step([dict(id=0, tokens=PROMPT[9:], want=[13])])
    last.attend = attend
    got = engine.step([dict(id=0, tokens=PROMPT[9:], want=[13])])[0]
    assert float((got.double() - want.double()).norm() / want.double().norm()) < 0.012
    engine.pool.release(0)
    assert paged.pages.free_pages() == 12
