"""GPU: the package's LLaMA with its keys and values in pages, behind the engine: against the LLaMA that caches one sequence, several requests at
once against each alone, 8-bit caches, a window with first tokens beyond the block size, and pages that come back."""
import json

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def llama(heads=4, width=128, layers=2, block=64, vocab=96, quantize="gptq.int4", seed=3):
    import lit_llama_b200 as P
    from lit_llama_b200.utils import quantization
    from oracle import llama_oracle as O

    sd = O.synth_state_dict(layers, heads, width, vocab, quantize, dtype=torch.bfloat16, seed=seed)
    prev = torch.get_default_dtype()
    torch.set_default_dtype(torch.bfloat16)
    try:
        with torch.device(DEV), quantization(quantize):
            model = P.LLaMA(P.LLaMAConfig(block_size=block, vocab_size=vocab, n_layer=layers, n_head=heads, n_embd=width))
    finally:
        torch.set_default_dtype(prev)
    model.load_state_dict(sd)
    return model.eval()


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


PROMPT = [3, 17, 40, 41, 2, 77, 5, 9, 33, 60, 8, 8, 1, 90, 14, 22, 7, 50, 31, 12, 66, 2, 4]


# Two layers, in each some eight roundings of the stream and of what is added to it to bf16 that the two paths do not share (2^-9 in the mean, independent), and
# the head's: 2^-9 sqrt(2 * 2 * 8 + 2) = 0.012 of the logits' norm.  An 8-bit cache: entries off by up to 2^-4 (e4m3) or 1 / 254 of the row's largest.
BOUND = {"act": 0.012, "int8": 0.03, "fp8": 0.08}


@pytest.mark.parametrize("store", ["act", "int8", "fp8"])
@pytest.mark.parametrize("portions", [[23], [1] * 23, [7, 1, 15]], ids=["prompt", "tokens", "portions"])
def test_logits_are_those_of_the_llama_with_one_sequence(store, portions):
    import lit_llama_b200 as P
    from lit_llama_b200.registry import LLaMASequenceModel

    model = llama()
    want = P.Engine(LLaMASequenceModel(model, 64), n_slots=1).step([dict(id=0, tokens=PROMPT, want=list(range(23)))])[0]
    engine = P.Engine(P.PagedLLaMAModel(model, pages=8, page=16, store=store), n_slots=2)
    at, got = 0, []
    for n in portions:
        got.append(engine.step([dict(id="r", tokens=PROMPT[at:at + n], want=list(range(n)))])[0])
        at += n
    assert rel(torch.cat(got), want) < BOUND[store]


def test_requests_together_get_what_each_gets_alone():
    import lit_llama_b200 as P

    model = llama()
    prompts = {"a": PROMPT, "b": PROMPT[5:9], "c": PROMPT[::-1] + PROMPT[:3]}
    alone = {}
    for r, p in prompts.items():
        engine = P.Engine(P.PagedLLaMAModel(model, pages=12, page=16), n_slots=1, prefill_chunk=9)
        engine.add_request(r, p, 12)
        alone.update(engine.run())
    paged = P.PagedLLaMAModel(model, pages=12, page=16)
    engine = P.Engine(paged, n_slots=2, prefill_chunk=9)                   # the third waits for a slot
    for r, p in prompts.items():
        engine.add_request(r, p, 12)
    assert engine.run() == alone
    assert paged.pages.free_pages() == 12                                   # all came back


def test_a_sequence_longer_than_the_block_keeps_its_window_and_first_tokens():
    import lit_llama_b200 as P

    model = llama(block=32)
    paged = P.PagedLLaMAModel(model, pages=6, page=16, window=24, first=2)
    engine = P.Engine(paged, n_slots=1, prefill_chunk=16)
    out = engine.generate(PROMPT, 150)
    assert len(out) == 23 + 150 and paged.pages.free_pages() == 6
    engine = P.Engine(P.PagedLLaMAModel(model, pages=6, page=16), n_slots=1, prefill_chunk=16)
    with pytest.raises(P.state.PoolFull):                                   # without a window the block size is the end
        engine.generate(PROMPT, 150)


def test_pages_that_run_out_and_slots_at_another_position():
    import lit_llama_b200 as P

    paged = P.PagedLLaMAModel(llama(), pages=2, page=16)
    engine = P.Engine(paged, n_slots=2)
    engine.step([dict(id="a", tokens=PROMPT[:20])])
    with pytest.raises(P.state.PoolFull):
        engine.step([dict(id="b", tokens=PROMPT[:20])])
    engine.step([dict(id="a", tokens=PROMPT[20:23])], end=["a"])
    assert paged.pages.free_pages() == 2
    ctx = P.mixers.StepContext(1, torch.tensor([0, 7], dtype=torch.int32, device=DEV), {}, torch.bfloat16, pos_hint=7, slot_hint=0)
    with pytest.raises(RuntimeError, match="position"):
        paged.forward_portion(torch.tensor([1], device=DEV), ctx)


def test_the_configuration_asks_for_pages(tmp_path):
    import lit_llama_b200 as P
    from lit_llama_b200.registry import LLaMASequenceModel

    model = llama()
    torch.save(model.state_dict(), tmp_path / "lit-llama.pth")
    config = dict(architecture="LLaMA", block_size=64, vocab_size=96, n_layer=2, n_head=4, n_embd=128, quantize="gptq.int4")
    (tmp_path / "config.json").write_text(json.dumps(config))
    assert isinstance(P.load_model(str(tmp_path)), LLaMASequenceModel)
    (tmp_path / "config.json").write_text(json.dumps(dict(config, kv_cache=dict(pages=8, page=16, store="int8"))))
    loaded = P.load_model(str(tmp_path))
    assert isinstance(loaded, P.PagedLLaMAModel) and loaded.caches[1].store == "int8"
    a = P.Engine(loaded, n_slots=1).generate(PROMPT, 8)
    b = P.Engine(P.PagedLLaMAModel(model, pages=8, page=16, store="int8"), n_slots=1).generate(PROMPT, 8)
    assert a == b
