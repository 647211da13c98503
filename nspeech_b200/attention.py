"""Attention through a sliding window with sinks (``nq_window_attention``).

The reference's decoders and Moonshine's encoder run it between the matmuls
(``flash_attention_fwd``, kernels/moonshine_kernels.py:749-845; sliding window
of src/moonshine/encoder.rs:116-135).  Of a sequence with n_q queries and n_k
keys, query i stands at position ``p = n_k - n_q + i`` and sees key j when
``j <= p + right`` and (``j >= p - left`` or ``j < sinks``); a negative left or
right is no limit.  ``nspeech_b200.cache`` runs the same over a paged cache.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import lib as _l
from .fast_matmul import MatMulError

_n = _l.native()


def _on(stream: torch.cuda.Stream, t: torch.Tensor):
    """The context of a call that is given a stream: everything it makes belongs to that stream."""
    if stream.device != t.device:
        raise MatMulError(f"the stream is on {stream.device}, the tensors on {t.device}")
    return torch.cuda.stream(stream)


def window_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, left: int = -1, right: int = -1, sinks: int = 0,
                     scale: Optional[float] = None, q_offsets: Optional[torch.Tensor] = None,
                     k_offsets: Optional[torch.Tensor] = None, q_lens: Optional[torch.Tensor] = None,
                     k_lens: Optional[torch.Tensor] = None, seqs: Optional[int] = None, out: Optional[torch.Tensor] = None,
                     stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Softmax attention of q [rows, q_heads, head_dim] over k, v [rows, kv_heads, head_dim] (f32 or bf16, any token and
    head strides); q_heads a multiple of kv_heads, head_dim up to 128, scale head_dim ** -0.5 unless given.

    Ragged batches: sequence b has the rows between ``q_offsets[b]`` and ``q_offsets[b + 1]`` (CUDA int32 [seqs + 1]),
    keys by ``k_offsets`` alike.  Without offsets each of `seqs` sequences (1 unless given) has as many rows.
    ``q_lens`` / ``k_lens`` (int32 [seqs]): only so many of a span's rows count, the others are padding.  Rows of no
    sequence are left as they are in `out`, which may be q itself and otherwise overlaps no input; a query that sees no key
    gives zeros, one that is NaN gives NaN.  There is no gradient: inputs that want one are refused unless gradients are
    off.  With `stream` the call runs as under ``torch.cuda.stream(stream)``."""
    if stream is not None:
        with _on(stream, q):
            return window_attention(q, k, v, left, right, sinks, scale, q_offsets, k_offsets, q_lens, k_lens, seqs, out)
    return _n.window_attention(q, k, v, left, right, sinks, scale, q_offsets, k_offsets, q_lens, k_lens, seqs, out)
