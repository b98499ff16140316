"""GPU: rows, queries and steps at the smallest sizes and off their 16-byte borders, through PagedCache."""
import pytest
import torch

from test_gpu_paged import DEV, IDS, TYPES, check, gen, make
from test_gpu_paged_rows import poison, step_of

pytestmark = pytest.mark.gpu


def same(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a._pool, b._pool) if x is not None)


def odd(x, how):
    """The same values: a slice of a wider product whose rows are no multiple of 16 bytes, off its border by one entry, transposed, or expanded."""
    rows, heads, size = x.shape
    wide = torch.zeros(rows, heads * size + 75, dtype=x.dtype, device=x.device)
    if how == "wide":
        wide[:, :heads * size] = x.reshape(rows, -1)
        return wide[:, :heads * size].unflatten(1, (heads, size))
    if how == "off":
        wide[:, 1:1 + heads * size] = x.reshape(rows, -1)
        return wide[:, 1:1 + heads * size].unflatten(1, (heads, size))
    if how == "heads":
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    if how == "entries":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    y = torch.zeros(rows, heads, size + 1, dtype=x.dtype, device=x.device)      # a column behind every head
    y[..., :size] = x
    return y[..., :size]


HOW = ["wide", "off", "heads", "entries", "columns"]


@pytest.mark.parametrize("dtype,store", TYPES, ids=IDS)
@pytest.mark.parametrize("how", HOW)
@pytest.mark.parametrize("heads,kv_heads,sequences", [(4, 4, [(1, 20)]), (1, 1, [(1, 20)]), (4, 2, [(5, 20), (2, 2)]), (1, 1, [(6, 20)]), (8, 2, [(40, 70)])])
def test_rows_of_every_stride(dtype, store, how, heads, kv_heads, sequences):
    cache, step, seqs = make(dtype, store, kv_heads, 32, 16, 16, sequences)
    other, _, _ = make(dtype, store, kv_heads, 32, 16, 16, sequences)
    g = gen(2)
    k, v, q = (torch.randn(step.rows, h, d, generator=g).to(dtype).to(DEV) for h, d in ((kv_heads, 32), (kv_heads, 16), (heads, 32)))
    before = [x.clone() for x in cache._pool if x is not None]
    a, b, c = odd(k, how), odd(v, how), odd(q, how)
    assert torch.equal(a, k) and torch.equal(b, v) and torch.equal(c, q)
    cache.write(k, v, step)
    assert any(not torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(before, (x for x in cache._pool if x is not None)))
    other.write(a, b, step)
    assert same(cache, other)
    got = cache.attend(q, step)
    assert torch.equal(cache.attend(c, step), got)
    check(got, q.cpu(), cache, seqs, 32 ** -0.5)


def test_one_row_of_many_as_a_slice():
    """The first row of a product's slice: torch calls it contiguous whatever its stride, which is no multiple of 16 bytes."""
    cache, step, seqs = make(torch.bfloat16, "act", 4, 32, 32, 16, [(1, 20)])
    wide = torch.randn(9, 475, generator=gen(1)).to(torch.bfloat16).to(DEV)
    x = wide[:, :128].view(9, 4, 32)[:1]
    assert x.is_contiguous() and x.stride(0) == 475
    cache.write(x, x, step)
    assert all(torch.equal(y, x) for y in cache.read(step))
    check(cache.attend(x, step), x.cpu(), cache, seqs, 32 ** -0.5)
    x = wide[3:4, 3:131].view(1, 4, 32)                      # and off its border
    cache.write(x, x, step)
    assert all(torch.equal(y, x) for y in cache.read(step))
    check(cache.attend(x, step), x.cpu(), cache, seqs, 32 ** -0.5)


@pytest.mark.parametrize("dtype,store", [TYPES[0], TYPES[1], TYPES[3]], ids=[IDS[0], IDS[1], IDS[3]])
def test_steps_without_rows(dtype, store):
    """No sequences, or sequences without new tokens: nothing is written, and the results are empty."""
    from lit_llama_b200 import PagePool

    cache, _, _ = make(dtype, store, 2, 64, 32, 16, [(1, 40)])
    before = [x.clone() for x in cache._pool if x is not None]
    pool = PagePool(8, 16, DEV)
    k, v, q = (torch.empty(0, h, d, dtype=dtype, device=DEV) for h, d in ((2, 64), (2, 32), (4, 64)))
    for entries in ([], [("a", 0)], [("a", 0), ("b", 0)]):
        step = pool.step(entries)
        cache.write(k, v, step)
        assert [tuple(x.shape) for x in cache.read(step)] == [(0, 2, 64), (0, 2, 32)]
        assert cache.attend(q, step).shape == (0, 4, 32)
        out = torch.empty(0, 4, 32, dtype=dtype, device=DEV)
        assert cache.attend(q, step, out=out) is out
    assert all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(before, (x for x in cache._pool if x is not None)))
    # rows behind a step without any
    some = torch.ones(3, 4, 64, dtype=dtype, device=DEV)
    cache.write(some[:, :2], some[:, :2, :32].contiguous(), step)
    poison((3, 4, 32), dtype=dtype)
    assert cache.attend(some, step).shape == (3, 4, 32) and not cache.attend(some, step).any()


@pytest.mark.parametrize("dtype,store", [TYPES[0], TYPES[1], TYPES[3]], ids=[IDS[0], IDS[1], IDS[3]])
def test_a_step_without_sequences_is_zeros(dtype, store):
    cache, _, _ = make(dtype, store, 2, 64, 32, 16, [(1, 40)])
    step = step_of([0], [], 6)
    poison((6, 4, 32), (6, 2, 64), (6, 2, 32), dtype=dtype)
    assert not cache.attend(torch.ones(6, 4, 64, dtype=dtype, device=DEV), step).any()
    assert not any(x.any() for x in cache.read(step))
