"""GPU: beam search's selection against the definition in 64 bits."""
import pytest
import torch

import tree_oracle as T

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32
INF = float("inf")


def check(logits, scores, count):
    """Beams and tokens are equal.  Values: a term e^d of a beam's sum is 2^(d log2 e), d = x - max rounded once (2^-24 of itself), times log2 e as f32 has it, rounded (2^-24
    each): off by 3 |d| 2^-24 of itself, and by 2^-22 for the power of two.  Over the sum |d| weighted with e^d is at most ln(vocab) < 12.3 (an entropy less what is not
    negative).  A thread's 32 terms are added in pairs, five roundings of 2^-24; all else is in 64 bits.  Together (37 + 4 + 5) 2^-24 of the sum, and its logarithm off by
    as much; the value is then rounded once, by 2^-24 of itself."""
    from lit_llama_b200 import beam_select

    values, beams, tokens = beam_select(logits, scores, count)
    for g in range(logits.shape[0]):
        v, b, t = T.select(logits[g], scores[g].cpu(), count)
        assert beams[g].tolist() == b.tolist() and tokens[g].tolist() == t.tolist(), g
        got = values[g].cpu().double()
        same = torch.isinf(v)
        assert torch.equal(got[same], v[same])
        assert bool(((got - v).abs()[~same] <= 2.0 ** -24 * v.abs()[~same] + 46 * 2.0 ** -24).all())
    return values, beams, tokens


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("groups,beams,vocab,count", [(1, 1, 1, 1), (1, 1, 5, 5), (2, 3, 7, 20), (1, 4, 32000, 8), (3, 8, 4099, 16), (48, 8, 8193, 16), (2, 16, 50257, 32), (1, 2, 2047, 1),
                                                      (5, 64, 300, 64), (1, 5, 130000, 64), (40, 16, 16390, 17), (0, 4, 100, 4)])
def test_selection(groups, beams, vocab, count, dtype):
    g = torch.Generator().manual_seed(groups + vocab)
    x = (torch.randn(groups, beams, vocab, generator=g) * 3).to(dtype).to(DEV)
    s = (-3 * torch.rand(groups, beams, generator=g)).to(DEV)
    check(x, s, count)


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("vocab", [40, 3000, 20000])
def test_ties_go_to_the_lowest_beam_and_token(vocab, dtype):
    """All logits alike, few different ones, the same beam twice."""
    g = torch.Generator().manual_seed(vocab)
    flat = torch.full((2, 4, vocab), 1.5)
    flat[1] = torch.randint(0, 3, (4, vocab), generator=g).float()
    flat[1, 2] = flat[1, 1]
    s = torch.tensor([[-1.0, -1.0, -2.0, -1.0], [-1.0, -1.5, -1.5, -9.0]], device=DEV)
    for count in (1, 16, 40, 64):
        check(flat.to(dtype).to(DEV), s, count)
    zeros = torch.zeros(1, 1, vocab)
    zeros[0, 0, ::2] = -0.0
    check(zeros.to(dtype).to(DEV), torch.zeros(1, 1, device=DEV), 30)


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("vocab", [12, 9000])
def test_beams_that_are_out(vocab, dtype):
    g = torch.Generator().manual_seed(7)
    x = torch.randn(8, 3, vocab, generator=g)
    s = -torch.rand(8, 3, generator=g)
    s[0, 1:] = -INF                                                        # the first step of a search: one beam
    s[1] = -INF
    x[2, 0, 5], x[2, 1, 3] = float("nan"), INF
    x[3, 1] = -INF
    x[4, :, 10:] = -INF                                                    # few tokens are allowed
    x[5, 0] = -INF
    x[5, 0, vocab - 1] = -1e30
    s[6, 2], s[6, 0] = INF, float("nan")
    x[7, 0] = float("nan")
    x[7, 1:] = -INF
    for count in (1, 8, 31, 36):
        check(x.to(dtype).to(DEV), s.to(DEV), min(count, 3 * vocab))


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
def test_logits_of_any_stride(dtype):
    """Rows that begin elsewhere within 16 bytes are shared among threads otherwise, so the sums' roundings differ: beams and tokens are the same, and values within the
    bound of `check`, which holds for every order of the terms in pairs."""
    from lit_llama_b200 import beam_select

    x = torch.randn(4, 6, 1001, device=DEV).to(dtype)
    s = -torch.rand(4, 6, device=DEV)
    want = check(x, s, 12)
    wide = torch.full((4, 6, 1040), 90.0, dtype=dtype, device=DEV)
    wide[..., 5:1006] = x
    apart = torch.full((4, 9, 1001), 90.0, dtype=dtype, device=DEV)
    apart[:, :6] = x
    for y in (wide[..., 5:1006], apart[:, :6], x.transpose(0, 1).contiguous().transpose(0, 1), x.transpose(1, 2).contiguous().transpose(1, 2), torch.cat([x.flatten()[:1], x.flatten()])[1:].view(4, 6, 1001)):
        assert all(torch.equal(a, b) for a, b in zip(check(y, s, 12)[1:], want[1:]))
    one = x[:1, :1].expand(3, 5, 1001)
    assert all(torch.equal(a, b) for a, b in zip(beam_select(one, s[:3, :5], 12), beam_select(one.contiguous(), s[:3, :5].contiguous(), 12)))
    assert all(torch.equal(a, b) for a, b in zip(beam_select(x[:, :1], s[:, :1], 3), beam_select(x[:, :1].contiguous(), s[:, :1].contiguous(), 3)))


def test_far_scores_and_logits():
    """Scores of long continuations, logits around large values: the order is that of 64 bits."""
    x = torch.randn(2, 4, 5000, device=DEV) * 0.01 + 1000.0
    check(x, torch.tensor([[-1e4, -1e4 - 0.001, -1e4 + 0.001, -2e4], [-1.0, -1.001, -1e30, 0.5]], device=DEV), 32)


def test_recorded_and_replayed():
    from lit_llama_b200 import beam_select

    x, s = torch.randn(3, 8, 9001, device=DEV), -torch.rand(3, 8, device=DEV)
    beam_select(x, s, 16)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):                                                     # two graphs, each with a work space of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = beam_select(x, s, 16)
        graphs.append((graph, got))
    for _ in range(3):
        x.normal_()
        want = [t.clone() for t in check(x, s, 16)]
        for graph, got in graphs:
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_refusals():
    from lit_llama_b200 import beam_select

    x, s = torch.zeros(2, 3, 10, device=DEV), torch.zeros(2, 3, device=DEV)
    for bad in (dict(logits=x[0]), dict(logits=x.half()), dict(logits=x[..., :0]), dict(scores=s[:, :2]), dict(scores=s.double()), dict(scores=s.cpu()), dict(count=0), dict(count=31),
                dict(count=65), dict(logits=torch.zeros(1, 65, 10, device=DEV), scores=torch.zeros(1, 65, device=DEV))):
        with pytest.raises(ValueError):
            beam_select(**dict(dict(logits=x, scores=s, count=4), **bad))
    with pytest.raises(RuntimeError, match="CUDA only"):
        beam_select(x.cpu(), s.cpu(), 4)
