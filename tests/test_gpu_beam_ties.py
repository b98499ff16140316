"""GPU: beam search's selection where values of different beams are equal or neighbours: their order is that of 64 bits, wherever a row begins."""
import pytest
import torch

import tree_oracle as T
from test_gpu_beam import BF, DEV, F32, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("vocab", [9, 1001, 4099, 8193, 50257, 100003])
@pytest.mark.parametrize("groups,beams,count", [(1, 8, 16), (3, 5, 33), (48, 8, 16), (1, 64, 64)])
def test_beams_alike(groups, beams, count, vocab, dtype):
    """The same logits in every beam of a group, in rows that begin anywhere within 16 bytes: equal scores tie to the lowest beam, others differ by a step of f32."""
    if groups * beams * vocab > 1 << 24:
        groups, beams = min(groups, 2), min(beams, 8)
    g = torch.Generator().manual_seed(vocab + groups)
    x = (torch.randn(groups, 1, vocab, generator=g) * 3).to(dtype).expand(groups, beams, vocab).contiguous().to(DEV)
    count = min(count, beams * vocab)
    check(x, torch.full((groups, beams), -1.25, device=DEV), count)
    steps = torch.randint(-3, 4, (groups, beams), generator=g)
    check(x, (-1.25 + steps * 2.0 ** -23).to(DEV), count)
    if groups == 1:                                                        # rows apart, in any alignment
        wide = torch.zeros(1, beams, vocab + 5, dtype=dtype, device=DEV)
        wide[..., 3:vocab + 3] = x
        check(wide[..., 3:vocab + 3], torch.full((1, beams), -1.25, device=DEV), count)


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("vocab", [1001, 8193, 32000, 100003])
def test_beams_whose_values_are_neighbours(vocab, dtype):
    """Beams of different logits whose scores put their largest values some 10^-9 to 10^-6 apart, in any order: less than the roundings of sums in f32."""
    g = torch.Generator().manual_seed(vocab)
    x = (torch.randn(4, 6, vocab, generator=g) * 2).to(dtype)
    x[2] = x[2, 0].roll(1, -1) if vocab == 1001 else torch.stack([x[2, 0].roll(97 * w, -1) for w in range(6)])      # the same sums but for their order
    top = torch.log_softmax(x.double(), -1).amax(-1)
    # scores near -top, small where they can be: f32 has them to 2^-26 or so; then every value is what the score as it is makes of it
    s = (-top - 1e-3 + torch.rand(4, 6, generator=g, dtype=torch.float64) * torch.tensor([1e-6, 1e-7, 1e-6, 3e-6])[:, None]).float()
    values = s.double() + top
    assert float((values.sort(-1).values.diff(dim=-1)).min()) >= 0.0
    gap = values.sort(-1).values.diff(dim=-1)
    apart = ((gap == 0.0) | (gap > 1e-12)).all(-1)                         # orders that 64 bits decide
    keep = [i for i in range(4) if bool(apart[i])]
    assert len(keep) >= 2
    check(x[keep].to(DEV), s[keep].to(DEV), 12)


def test_neighbours_around_the_last_place():
    """Which of the beams' equal or nearly equal values are chosen at all: many for the last places, more than the list of candidates holds."""
    vocab = 3001
    x = torch.zeros(1, 64, vocab)
    x[..., ::7] = 1.0
    s = -torch.arange(64, dtype=torch.float32) % 5 * 2.0 ** -22 - 0.5
    for dtype in (BF, F32):
        for count in (1, 7, 40, 64):
            check(x.to(dtype).to(DEV), s[None].to(DEV), count)
            check(x.to(dtype).to(DEV)[:, :3], s[None, :3].to(DEV), count)
    hidden = torch.full((1, 64, vocab), float("-inf"))
    hidden[0, :, 5] = 2.0
    for count in (3, 64):
        check(hidden.to(DEV), s[None].to(DEV), count)
        check(hidden.to(BF).to(DEV), torch.full((1, 64), -2.0, device=DEV), count)


def test_what_is_given_repeats_itself():
    g = torch.Generator().manual_seed(3)
    from lit_llama_b200 import beam_select

    x, s = torch.randn(12, 8, 50257, generator=g).to(BF).to(DEV), (-torch.rand(12, 8, generator=g)).to(DEV)
    x[3] = x[3, :1]
    s[3] = -0.5
    once = beam_select(x, s, 16)
    assert [int(b) for b in once[1][3]] == T.select(x[3], s[3], 16)[1].tolist()
    for _ in range(20):
        assert all(torch.equal(a, b) for a, b in zip(beam_select(x, s, 16), once))


@pytest.mark.parametrize("dtype", [BF, F32], ids=str)
@pytest.mark.parametrize("vocab", [7, 500, 4097, 32000])
def test_scores_that_make_up_for_logits(vocab, dtype):
    """The same logits, in eighths, with scores that are eighths too: many tokens of different beams have the same value, which is that of sums without a rounding."""
    from lit_llama_b200 import beam_select

    g = torch.Generator().manual_seed(vocab)
    x = (torch.randint(-40, 40, (8, 1, vocab), generator=g) / 8).to(dtype)
    for _ in range(8):
        s = -torch.randint(0, 40, (8, 6), generator=g) / 8
        sums = (s[..., None] + x.float()).flatten(1)                       # exact; a group's beams have one logarithm
        at = torch.sort(sums, dim=-1, descending=True, stable=True).indices[:, :32]
        values, beams, tokens = beam_select(x.expand(8, 6, vocab).contiguous().to(DEV), s.to(DEV), min(32, 6 * vocab))
        assert torch.equal(beams.cpu().long() * vocab + tokens.cpu(), at)
