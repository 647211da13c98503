"""Beam search over the decoder's logits (``nq_beam_select``, ``nq_beam_reorder``).

One step takes the lm_head's logits of all beams, picks the best continuations by log probability, and says for each
which row it comes from, so that ``PagedCache.fork`` and ``beam_reorder`` bring the beams' pages and recurrent states
along.  One beam is greedy decoding (the reference's ``argmax_logits``, src/moonshine/gpu_decoder_metal.rs:110-243).  A
transducer's search over tokens, durations and blanks (``beam_decode``, src/parakeet/transducer.rs:1116) is another one.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from . import lib as _l
from .attention import _on

_n = _l.native()


def beam_select(logits: torch.Tensor, scores: torch.Tensor, finished: Optional[torch.Tensor] = None, eos: int = -1,
                out: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]] = None,
                stream: Optional[torch.cuda.Stream] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The best `beams` continuations of each item: (scores f32, parents int32, tokens int32, finished bool), each
    [items, beams], best first, equal scores by lower beam, then lower token.

    logits [items, beams, vocab] (f32 or bf16), scores f32 [items, beams] (sums of log probabilities; -inf for beams that
    do not exist yet), finished bool [items, beams]: a finished beam goes on only as itself, with token `eos` and its
    score unchanged.  parents are rows of all items' beams (item * beams + beam).  Up to 32 beams.  Rows may lie any even
    distance apart (a padded lm_head).  `out` may hold the inputs of the same kind; otherwise outputs overlap nothing."""
    if stream is not None:
        with _on(stream, logits):
            return beam_select(logits, scores, finished, eos, out)
    return _n.beam_select(logits, scores, finished, eos, out)


def beam_reorder(states: Sequence[torch.Tensor], parents: torch.Tensor, out: Optional[Sequence[torch.Tensor]] = None,
                 stream: Optional[torch.cuda.Stream] = None) -> List[torch.Tensor]:
    """out[i][r] = states[i][parents[r]] for every state (any dtype, [rows, ...] with contiguous rows), in one launch for
    up to 16 states.  parents: int32, `rows` of them in any shape (``beam_select``'s); one out of range stands for the row
    itself.  out[i] may be states[i], but overlaps no other state or output, nor parents."""
    if stream is not None:
        with _on(stream, parents):
            return beam_reorder(states, parents, out)
    return _n.beam_reorder(states, parents, out)
