"""Beam search's selection, beside the sampling of generate.py."""
from functools import lru_cache
from typing import Tuple

import torch

from . import _seqlib as S
from .paged import ACTS, _launch

MOST, MOST_VOCAB = 64, 1 << 30


def beam_select(logits: torch.Tensor, scores: torch.Tensor, count: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The `count` most likely continuations of every group of beams by a token:

        value[g, w, v] = scores[g, w] + logits[g, w, v] - log sum_u exp logits[g, w, u]

    logits [groups, beams, vocab] (bf16 or f32, rows of any stride), scores f32 [groups, beams] (of what the beams have so far; -inf: a beam that is out).  Returns, [groups,
    count] each and the largest first, the values (f32), the beams that they continue and the tokens (int32).  Ties go to the lowest beam, then the lowest
    token; the order is that of the values in 64 bits, before they are rounded to f32 (beams whose values are within some 5e-6 have their sums formed again for that, 30 us for a row
    of 100003 tokens).  A beam is out too, its values -inf, where a logit is NaN or +inf or none is above -inf.
    At most 64 beams and 64 continuations.  One kernel pass over the logits and one over what is left (include/b2l_seq.h); CUDA only, no derivatives."""
    shape, device = logits.shape, logits.device
    if len(shape) != 3 or logits.dtype not in ACTS or shape[1] < 1 or shape[2] < 1:
        raise ValueError(f"beam selection: logits {tuple(shape)} {logits.dtype}: [groups, beams, vocab] in bf16 or f32")
    groups, beams, vocab = shape
    if scores.shape != shape[:2] or scores.dtype != torch.float32 or scores.device != device:
        raise ValueError(f"beam selection: scores {tuple(scores.shape)} {scores.dtype} on {scores.device}: {(groups, beams)} f32 on {device}")
    count = int(count)
    if not 0 < count <= min(MOST, beams * vocab) or beams > MOST or vocab >= MOST_VOCAB:
        raise ValueError(f"beam selection: {count} of {beams} beams and {vocab} tokens: at most {MOST} beams and {MOST} of them, fewer than {MOST_VOCAB} tokens")
    # rows at equal distances, their entries consecutive; strides of a single row, beam or group are whatever torch says
    s0, s1, s2 = logits.stride()
    ld = s1 if beams > 1 else s0 if groups > 1 else vocab
    if (s2 != 1 and vocab > 1) or ld < vocab or (groups > 1 and beams > 1 and s0 != beams * s1):
        logits, ld = logits.contiguous(), vocab
    if not scores.is_contiguous():
        scores = scores.contiguous()
    size = _work(groups, beams, vocab, count, logits.dtype, device.index)
    values, of, tokens = scores.new_empty((3, groups, count), dtype=torch.int32).unbind(0)
    values, work = values.view(torch.float32), scores.new_empty(-(-size // 4))
    _launch(device, "b2l_seq_beam_select", logits.data_ptr(), ld, scores.data_ptr(), values.data_ptr(), of.data_ptr(), tokens.data_ptr(), work.data_ptr(), size, groups, beams, vocab, count,
            S.act_code(logits.dtype))
    return values, of, tokens


@lru_cache(maxsize=256)
def _work(groups: int, beams: int, vocab: int, count: int, dtype: torch.dtype, device) -> int:
    """Bytes of work space: by the device too, whose SMs decide how rows are split."""
    if device is None:
        return 0                                                            # refused by the launch
    with torch.cuda.device(device):
        return S.lib().b2l_seq_beam_work(groups, beams, vocab, count, S.act_code(dtype))
