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
from .attention import _code, _device, _ints, _stream
from .fast_matmul import MatMulError


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(items: int, beams: int, vocab: int) -> int:
    n = _l.load().nq_beam_workspace(items, beams, vocab)
    if n < 0:
        _l.check(int(n))
    return n


_FLAGS = (torch.bool, torch.uint8)


def _pair(t: torch.Tensor, name: str, shape, dtypes, index: int) -> int:
    if t.shape != shape or t.dtype not in dtypes or t.get_device() != index or not t.is_contiguous():
        raise MatMulError(f"{name} must be contiguous {list(shape)} of {' or '.join(str(d) for d in dtypes)} on cuda:{index}")
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
    by = logits.stride()
    if vocab > 1 and by[2] != 1 or items > 1 and by[0] != beams * by[1]:
        raise MatMulError("logits must have unit stride along the vocabulary and evenly spaced rows")
    code, dev = _code(logits, "logits"), _device(logits, "logits")
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return beam_select(logits, scores, finished, eos, out, stream)
    pair = (items, beams)
    need = _workspace_bytes(items, beams, vocab)
    p_scores = _pair(scores, "scores", pair, (torch.float32,), dev)
    p_finished = _pair(finished, "finished", pair, _FLAGS, dev) if finished is not None else None
    if out is None:
        n = items * beams
        # one allocation for the outputs and the workspace: three rows of 32-bit words, the flags, then 8-byte entries
        at = (13 * n + 7) // 8 * 8
        buf = torch.empty(at + need, dtype=torch.uint8, device=logits.device)
        words = buf[:12 * n].view(torch.int32).view(3, items, beams)
        out = words[0].view(torch.float32), words[1], words[2], buf[12 * n:13 * n].view(torch.bool).view(items, beams)
        base = buf.data_ptr()
        p_out, p_ws, made = (base, base + 4 * n, base + 8 * n, base + 12 * n), base + at, buf
    else:
        p_out = [_pair(t, f"out[{i}]", pair, d, dev) for i, (t, d) in enumerate(zip(out, ((torch.float32,), (torch.int32,),
                                                                                         (torch.int32,), _FLAGS)))]
        made = torch.empty(need, dtype=torch.uint8, device=logits.device)
        p_ws = made.data_ptr()
    rc = _l.load().nq_beam_select(logits.data_ptr(), code, by[1] if beams > 1 else by[0] if items > 1 else vocab, items, beams, vocab,
                                  p_scores, p_finished, eos, *p_out, p_ws, need, _stream(dev, stream, made))
    if rc:
        _l.check(rc)
    return out


def beam_reorder(states: Sequence[torch.Tensor], parents: torch.Tensor, out: Optional[Sequence[torch.Tensor]] = None,
                 stream: Optional[torch.cuda.Stream] = None) -> List[torch.Tensor]:
    """out[i][r] = states[i][parents[r]] for every state (any dtype, [rows, ...] with contiguous rows), in one launch for
    up to 16 states.  parents: int32, `rows` of them in any shape (``beam_select``'s).  out[i] may be states[i]."""
    if not states:
        return []
    rows, dev = parents.numel(), _device(parents, "parents")
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return beam_reorder(states, parents, out, stream)
    ptr = _ints(parents.view(-1) if parents.is_contiguous() else parents, "parents", rows, dev)
    made = out is None
    out = [torch.empty_like(t, memory_format=torch.contiguous_format) for t in states] if made else list(out)
    if len(out) != len(states):
        raise MatMulError(f"{len(out)} outputs for {len(states)} states")
    src, dst, size, src_by, dst_by = [], [], [], [], []
    for t, o in zip(states, out):
        shape = t.shape
        if not shape or shape[0] != rows or t.get_device() != dev or o.get_device() != dev or o.dtype != t.dtype or o.shape != shape:
            raise MatMulError(f"a state must be [{rows}, ...] on cuda:{dev}, like its output")
        n = t.numel()
        if n == 0:
            continue
        each = t.element_size()
        row = n // rows * each
        by = []
        for x in (t, o):
            if x.is_contiguous():
                by.append(row)
            elif x[0].is_contiguous():
                by.append(x.stride(0) * each if rows > 1 else row)
            else:
                raise MatMulError("a state's rows must be contiguous")
        src.append(t.data_ptr())
        dst.append(o.data_ptr())
        size.append(row)
        src_by.append(by[0])
        dst_by.append(by[1])
    s = _stream(dev, stream, *(out if made else ()))
    for i in range(0, len(src), 16):
        m = min(16, len(src) - i)
        a = (ctypes.c_int64 * (5 * m))(*src[i:i + m], *dst[i:i + m], *size[i:i + m], *src_by[i:i + m], *dst_by[i:i + m])
        rc = _l.load().nq_beam_reorder(a, ctypes.byref(a, 8 * m), ctypes.byref(a, 16 * m), ctypes.byref(a, 24 * m),
                                       ctypes.byref(a, 32 * m), m, rows, ptr, s)
        if rc:
            _l.check(rc)
    return out
