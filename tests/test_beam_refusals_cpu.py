"""CPU: vocabularies of which a place in a row, or behind its last part, would not fit 32 bits are refused before anything is launched."""
import pytest
import torch

from lit_llama_b200 import _seqlib as S
from lit_llama_b200 import beam_select


@pytest.mark.parametrize("vocab", [1 << 30, (1 << 31) - 20000, (1 << 31) - 1])
@pytest.mark.parametrize("act", [0, 1])
def test_vocabularies_beyond_the_kernels_integers(vocab, act):
    lib = S.lib()
    assert lib.b2l_seq_beam_work(1, 1, vocab, 4, act) >= 0
    assert lib.b2l_seq_beam_select(64, vocab, 64, 64, 64, 64, 64, 1 << 40, 1, 1, vocab, 4, act, None) < 0
    assert b"tokens" in lib.b2l_seq_last_error()
    x = torch.zeros(1, dtype=torch.float32 if act else torch.bfloat16).expand(1, 1, vocab)
    with pytest.raises(ValueError, match="tokens"):
        beam_select(x, torch.zeros(1, 1), 4)
