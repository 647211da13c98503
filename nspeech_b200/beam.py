"""Beam search over the decoder's logits (``nq_beam_select``, ``nq_beam_reorder``).

One step takes the lm_head's logits of all beams, picks the best continuations by log probability, and says for each
which row it comes from, so that ``PagedCache.fork`` and ``beam_reorder`` bring the beams' pages and recurrent states
along.  One beam is greedy decoding (the reference's ``argmax_logits``, src/moonshine/gpu_decoder_metal.rs:110-243;
its beam search is ``beam_decode``, src/parakeet/transducer.rs:1116).
"""
from __future__ import annotations

import ctypes
import functools
from typing import List, Optional, Sequence, Tuple

import torch

from . import lib as _l
from .attention import _code, _here, _ints, _stream
from .fast_matmul import MatMulError


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(items: int, beams: int, vocab: int) -> int:
    n = _l.load().nq_beam_workspace(items, beams, vocab)
    if n < 0:
        _l.check(int(n))
    return n


def _pair(t: Optional[torch.Tensor], name: str, shape, dtypes, device) -> Optional[int]:
    if t is None:
        return None
    if tuple(t.shape) != shape or t.dtype not in dtypes or t.device != device or not t.is_contiguous():
        raise MatMulError(f"{name} must be contiguous {list(shape)} of {' or '.join(str(d) for d in dtypes)} on {device}")
    return t.data_ptr()


def beam_select(logits: torch.Tensor, scores: torch.Tensor, finished: Optional[torch.Tensor] = None, eos: int = -1,
                out: Optional[Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]] = None,
                stream: Optional[torch.cuda.Stream] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """The best `beams` continuations of each item: (scores f32, parents int32, tokens int32, finished bool), each
    [items, beams], best first, equal scores by lower beam, then lower token.

    logits [items, beams, vocab] (f32 or bf16), scores f32 [items, beams] (sums of log probabilities; -inf for beams that
    do not exist yet), finished bool [items, beams]: a finished beam goes on only as itself, with token `eos` and its
    score unchanged.  parents are rows of all items' beams (item * beams + beam).  Up to 32 beams."""
    if logits.dim() != 3:
        raise MatMulError("logits must be [items, beams, vocab]")
    items, beams, vocab = logits.shape
    code, dev = _code(logits, "logits"), logits.device
    if vocab > 1 and logits.stride(2) != 1 or items > 1 and logits.stride(0) != beams * logits.stride(1):
        raise MatMulError("logits must have unit stride along the vocabulary and evenly spaced rows")
    ld = logits.stride(1) if beams > 1 else logits.stride(0) if items > 1 else vocab
    pair, flags = (items, beams), (torch.bool, torch.uint8)
    with _here(logits, "logits"):
        need = _workspace_bytes(items, beams, vocab)
        if out is None:
            out = (torch.empty(pair, dtype=torch.float32, device=dev), torch.empty(pair, dtype=torch.int32, device=dev),
                   torch.empty(pair, dtype=torch.int32, device=dev), torch.empty(pair, dtype=torch.bool, device=dev))
        ptrs = (_pair(scores, "scores", pair, (torch.float32,), dev), _pair(finished, "finished", pair, flags, dev))
        outs = [_pair(t, n, pair, d, dev) for t, n, d in zip(out, ("out scores", "out parents", "out tokens", "out finished"),
                                                             ((torch.float32,), (torch.int32,), (torch.int32,), flags))]
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
        s = _stream(logits, stream, ws, *out)
        _l.check(_l.load().nq_beam_select(logits.data_ptr(), code, ld, items, beams, vocab, ptrs[0], ptrs[1], eos, *outs,
                                          ws.data_ptr(), need, s))
    return out


def beam_reorder(states: Sequence[torch.Tensor], parents: torch.Tensor, out: Optional[Sequence[torch.Tensor]] = None,
                 stream: Optional[torch.cuda.Stream] = None) -> List[torch.Tensor]:
    """out[i][r] = states[i][parents[r]] for every state (any dtype, [rows, ...] with contiguous rows), in one launch for
    up to 16 states.  parents: int32, `rows` of them in any shape (``beam_select``'s).  out[i] may be states[i]."""
    states = list(states)
    if not states:
        return []
    rows, dev = parents.numel(), parents.device
    ptr = _ints(parents.reshape(-1) if parents.is_contiguous() else parents, "parents", rows, dev)
    with _here(parents, "parents"):
        made = out is None
        out = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in states] if made else list(out)
        if len(out) != len(states):
            raise MatMulError(f"{len(out)} outputs for {len(states)} states")
        for t, o in zip(states, out):
            for x in (t, o):
                if x.dim() < 1 or x.shape[0] != rows or x.device != dev or x.dtype != t.dtype or x.shape != t.shape:
                    raise MatMulError(f"a state must be [{rows}, ...] on {dev}, like its output")
                if rows and not x[0].is_contiguous():
                    raise MatMulError("a state's rows must be contiguous")
        size = [t.numel() // rows * t.element_size() if rows else 0 for t in states]
        s = _stream(parents, stream, *(out if made else ()))
        for i in range(0, len(states), 16):
            part = [j for j in range(i, min(i + 16, len(states))) if size[j]]
            m = len(part)
            P, I = ctypes.c_void_p * m, ctypes.c_int64 * m
            stride = [[x[j].stride(0) * x[j].element_size() if rows > 1 else size[j] for j in part] for x in (states, out)]
            _l.check(_l.load().nq_beam_reorder(P(*(states[j].data_ptr() for j in part)), P(*(out[j].data_ptr() for j in part)),
                                               I(*(size[j] for j in part)), I(*stride[0]), I(*stride[1]), m, rows, ptr, s))
    return out
