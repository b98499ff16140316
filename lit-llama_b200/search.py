"""Beam search's selection, beside the sampling of generate.py."""
from typing import Tuple

import torch

from . import _seqlib as S
from .paged import _launch

MOST = 64


def beam_select(logits: torch.Tensor, scores: torch.Tensor, count: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The `count` most likely continuations of every group of beams by a token:

        value[g, w, v] = scores[g, w] + logits[g, w, v] - log sum_u exp logits[g, w, u]

    logits [groups, beams, vocab] (bf16 or f32, rows of any stride), scores f32 [groups, beams] (of what the beams have so far; -inf: a beam that is out).  Returns, [groups,
    count] each and the largest first, the values (f32), the beams that they continue and the tokens (int32).  Ties go to the lowest beam, then the lowest
    token; the order is that of the values before they are rounded to f32.  A beam is out too, its values -inf, where a logit is NaN or +inf or none is above -inf.
    At most 64 beams and 64 continuations.  One kernel pass over the logits and one over what is left (include/b2l_seq.h); CUDA only, no derivatives."""
    if logits.dim() != 3 or logits.dtype not in (torch.bfloat16, torch.float32) or logits.shape[1] < 1 or logits.shape[2] < 1:
        raise ValueError(f"beam selection: logits {tuple(logits.shape)} {logits.dtype}: [groups, beams, vocab] in bf16 or f32")
    groups, beams, vocab = logits.shape
    if scores.shape != (groups, beams) or scores.dtype != torch.float32 or scores.device != logits.device:
        raise ValueError(f"beam selection: scores {tuple(scores.shape)} {scores.dtype} on {scores.device}: {(groups, beams)} f32 on {logits.device}")
    count = int(count)
    if not 0 < count <= min(MOST, beams * vocab) or beams > MOST:
        raise ValueError(f"beam selection: {count} of {beams} beams and {vocab} tokens: at most {MOST} beams and {MOST} of them")
    rows = groups * beams
    s0, s1, s2 = logits.stride()
    if vocab > 1 and s2 != 1 or beams > 1 and s1 < vocab or groups > 1 and s0 != beams * (s1 if beams > 1 else s0 // beams) or (groups > 1 and beams == 1 and s0 < vocab):
        logits = logits.contiguous()
        s0, s1, s2 = logits.stride()
    ld = s1 if beams > 1 else s0 if groups > 1 else vocab
    scores = scores.contiguous()
    values = torch.empty((groups, count), dtype=torch.float32, device=logits.device)
    chosen = torch.empty((2, groups, count), dtype=torch.int32, device=logits.device)
    size = S.lib().b2l_seq_beam_work(groups, beams, vocab, count)
    work = torch.empty((size,), dtype=torch.uint8, device=logits.device)
    _launch(logits.device, "b2l_seq_beam_select", logits.data_ptr(), ld, scores.data_ptr(), values.data_ptr(), chosen[0].data_ptr(), chosen[1].data_ptr(), work.data_ptr(), size, groups,
            beams, vocab, count, S.act_code(logits.dtype))
    return values, chosen[0], chosen[1]
