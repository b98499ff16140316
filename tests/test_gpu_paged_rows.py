"""GPU: rows of no sequence.  A step's tensors may cover fewer rows than the host says (a step padded for a recording, tensors that were overwritten between
replays): what `attend` and `read` return for the others is zeros, not what the memory held before, and a given `out` keeps them."""
import pytest
import torch

import paged_oracle as O
from test_gpu_paged import DEV, IDS, TYPES, check, gen, make

pytestmark = pytest.mark.gpu


def step_of(starts, seqs, rows, **hints):
    """A step of [(new, length, pages)] whose rows begin at starts[0], with `rows` rows by the host's word."""
    from lit_llama_b200 import PagedStep

    width = max([1] + [len(p) for _, _, p in seqs])
    i32 = dict(dtype=torch.int32, device=DEV)
    table = torch.tensor([list(p) + [-1] * (width - len(p)) for _, _, p in seqs], **i32).view(len(seqs), width)
    return PagedStep(torch.tensor(starts, **i32), torch.tensor([m for _, m, _ in seqs], **i32), table, rows=rows, **hints)


def poison(*shapes, dtype):
    """Memory of these sizes, taken up again by the next tensors of them, is full of NaN."""
    torch.cuda.empty_cache()
    held = [torch.full(s, float("nan"), dtype=dtype, device=DEV) for s in shapes for _ in range(3)]
    del held


# heads, kv heads, sequences, rows before the first and behind the last, what the host says: the forms of single tokens (whole, in parts), of chunks (cut among
# the SMs or not) and both together
FORMS = {
    "tokens": (8, 2, [(1, 40), (1, 1), (0, 7), (1, 129)], 0, 5, {}),
    "tokens-before": (8, 2, [(1, 40), (0, 3), (1, 129)], 3, 2, dict(max_new=1, max_length=129)),
    "parts": (4, 2, [(1, 3000), (1, 2500)], 2, 3, dict(max_new=1, max_length=3000)),
    "empty-ends": (4, 2, [(0, 9), (1, 33), (0, 50)], 1, 4, {}),
    "chunk": (8, 2, [(40, 100), (130, 200)], 7, 30, {}),
    "chunk-in-parts": (8, 2, [(300, 4000)], 5, 91, dict(max_new=300, max_length=4000)),
    "both": (12, 4, [(1 + i % 4, 9000 - 100 * i) for i in range(60)] + [(200, 300)], 4, 60, dict(max_new=200, max_length=9000)),
}


@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
@pytest.mark.parametrize("form", FORMS)
def test_rows_of_no_sequence_are_zeros(dtype, store, form):
    heads, kv_heads, sequences, before, behind, hints = FORMS[form]
    cache, _, seqs = make(dtype, store, kv_heads, 64, 32, 16, sequences)
    starts = [before]
    for n, _, _ in seqs:
        starts.append(starts[-1] + n)
    rows = starts[-1] + behind
    step = step_of(starts, seqs, rows, **hints)
    q = torch.randn(rows, heads, 64, generator=gen(5)).to(dtype)
    qd = q.to(DEV)
    poison((rows, heads, 32), dtype=dtype)
    got = cache.attend(qd, step)
    assert not got[:before].any() and not got[starts[-1]:].any()
    if form != "both":                                                       # (compared with the restatement elsewhere)
        check(got[before:starts[-1]], q[before:starts[-1]], cache, seqs, 0.125)
    out = torch.full((rows, heads, 32), 7.0, dtype=dtype, device=DEV)
    cache.attend(qd, step, out=out)
    assert (out[:before] == 7.0).all() and (out[starts[-1]:] == 7.0).all() and torch.equal(out[before:starts[-1]], got[before:starts[-1]])
    poison((rows, kv_heads, 64), (rows, kv_heads, 32), dtype=dtype)
    for name, back in zip("kv", cache.read(step)):
        assert not back[:before].any() and not back[starts[-1]:].any()
        at, pool = O.places(seqs, 16), O.values(cache, name)
        want = torch.stack([pool[pg, :, i] for _, _, pg, i in at])
        del pool
        assert torch.equal(back[before:starts[-1]].cpu(), want.to(dtype))


@pytest.mark.parametrize("new,heads", [(1, 4), (64, 8)])
@pytest.mark.parametrize("dtype,store", [TYPES[0], TYPES[2], TYPES[3]], ids=[IDS[0], IDS[2], IDS[3]])
def test_a_recorded_step_that_covers_fewer_rows_later(dtype, store, new, heads):
    """Four places for sequences, recorded with all of them and replayed with two: the others' rows are zeros, not the last replay's results."""
    cache, _, seqs = make(dtype, store, 2, 64, 32, 16, [(new, 100 + 30 * b) for b in range(4)])
    rows = 4 * new
    step = step_of([0, new, 2 * new, 3 * new, rows], seqs, rows, max_new=new, max_length=200)
    q = torch.randn(rows, heads, 64, generator=gen(5)).to(dtype)
    qd = q.to(DEV)
    cache.attend(qd, step)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out, back = cache.attend(qd, step), cache.read(step)
    graph.replay()
    torch.cuda.synchronize()
    check(out, q, cache, seqs, 0.125)
    step.starts.copy_(torch.tensor([0, new, 2 * new, 2 * new, 2 * new], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    check(out[:2 * new], q[:2 * new], cache, seqs[:2], 0.125)
    assert not any(x[2 * new:].any() for x in (out, *back))


@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
def test_windows_beyond_every_position(dtype, store):
    """At positions below zero as well, where window and position together leave 32 bits; through the C entry itself, too."""
    cache, step, seqs = make(dtype, store, 2, 64, 64, 16, [(40, 40), (300, 300), (1, 1), (200, 900)])
    step.lengths.copy_(torch.tensor([7, 10, 0, 100], dtype=torch.int32))
    q = torch.randn(step.rows, 8, 64, generator=gen(3)).to(dtype).to(DEV)
    whole = cache.attend(q, step)
    assert whole.any()
    for window, first in ((16 * step.table.shape[1], 0), (2 ** 31 - 1, 0), (2 ** 31 - 1, 9), (2 ** 31, 0), (2 ** 32 + 5, 0), (3, 2 ** 31 - 1), (3, 2 ** 35)):
        assert torch.equal(cache.attend(q, step, window=window, first=first), whole)
    from lit_llama_b200 import _seqlib as S

    for window, first in ((2 ** 31 - 1, 0), (2 ** 31 - 1, 2 ** 31 - 1), (3, 2 ** 31 - 1)):
        sizes = (8, 2, 64, 64, window, first)
        codes = (step.max_new, step.max_length) + cache._codes
        floats = S.lib().b2l_seq_paged_attention_work(step.rows, step.seqs, step.table.shape[1], 16, *sizes, *codes)
        work, out = torch.empty(max(floats, 1), device=DEV), torch.zeros_like(whole)
        S.check(S.lib().b2l_seq_paged_attention(q.data_ptr(), 512, 64, *cache._at, *step._at, out.data_ptr(), work.data_ptr(), floats, step.rows, step.seqs, cache.n_pages, 16, *sizes,
                                                0.125, *codes, S.stream_ptr()), "b2l_seq_paged_attention")
        assert torch.equal(out, whole)
