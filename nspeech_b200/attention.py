"""Attention through a sliding window with sinks (``nq_window_attention``).

The reference's decoders and Moonshine's encoder run it between the matmuls
(``flash_attention_fwd``, kernels/moonshine_kernels.py:749-845; sliding window
of src/moonshine/encoder.rs:116-135).  Of a sequence with n_q queries and n_k
keys, query i stands at position ``p = n_k - n_q + i`` and sees key j when
``j <= p + right`` and (``j >= p - left`` or ``j < sinks``); a negative left or
right is no limit.  ``nspeech_b200.cache`` runs the same over a paged cache.
"""
from __future__ import annotations

import contextlib
import ctypes
import functools
from typing import Optional

import torch

from . import lib as _l
from .fast_matmul import MatMulError

_CODES = {torch.float32: _l.NQ_F32, torch.bfloat16: _l.NQ_BF16}


def _code(t: torch.Tensor, name: str) -> int:
    code = _CODES.get(t.dtype)
    if code is None:
        raise MatMulError(f"{name} has dtype {t.dtype} (f32 or bf16)")
    return code


def _here(t: torch.Tensor, name: str):
    """The tensor's device made ready, as a context in which it is the current one."""
    if not t.is_cuda:
        raise MatMulError(f"{name} must live on a CUDA device")
    index, now = t.device.index, torch.cuda.current_device()
    if index not in _l._inited:
        _l.init(index)
        torch.cuda.set_device(now)
    return contextlib.nullcontext() if index == now else torch.cuda.device(index)


def _stream(t: torch.Tensor, stream: Optional[torch.cuda.Stream], *made: Optional[torch.Tensor]) -> int:
    """The stream to launch on: `stream`, or the current one of t's device.  Tensors made for the call on the current
    stream are kept from reuse until `stream` is through with them."""
    if stream is None:
        return torch.cuda.current_stream(t.device).cuda_stream
    if stream.device != t.device:
        raise MatMulError(f"the stream is on {stream.device}, the tensors on {t.device}")
    for m in made:
        if m is not None:
            m.record_stream(stream)
    return stream.cuda_stream


def _rows(t: torch.Tensor, name: str, dtype: torch.dtype, device: torch.device) -> _l.Rows:
    if t.dim() != 3 or t.dtype != dtype or t.device != device or (t.stride(2) != 1 and t.shape[2] > 1 and t.numel()):
        raise MatMulError(f"{name} must be [rows, heads, head_dim] of {dtype} on {device} with unit last stride")
    return _l.Rows(t.data_ptr(), t.stride(0), t.stride(1))


def _ints(t: Optional[torch.Tensor], name: str, n: Optional[int], device: torch.device) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous() or t.device != device or (n is not None and t.numel() != n):
        raise MatMulError(f"{name} must be contiguous int32{'' if n is None else f' [{n}]'} on {device}")
    return t.data_ptr()


def _output(out: Optional[torch.Tensor], q: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if out.shape != q.shape:
        raise MatMulError(f"out has shape {tuple(out.shape)}, q {tuple(q.shape)}")
    return out


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(*sizes) -> int:
    n = _l.load().nq_window_attention_workspace(*sizes)
    if n < 0:
        _l.check(int(n))
    return n


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
    sequence are left as they are in `out`; a query that sees no key gives zeros."""
    if q.dim() != 3 or k.dim() != 3 or v.dim() != 3:
        raise MatMulError("q, k and v must be [rows, heads, head_dim]")
    if k.shape != v.shape or q.shape[2] != k.shape[2] or q.shape[1] % max(1, k.shape[1]):
        raise MatMulError(f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit together")
    code, dev = _code(q, "q"), q.device
    with _here(q, "q"):
        if seqs is None:
            seqs = next((t.numel() - d for t, d in ((q_offsets, 1), (k_offsets, 1), (q_lens, 0), (k_lens, 0)) if t is not None), 1)
        out = _output(out, q)
        rows = [_rows(t, n, q.dtype, dev) for t, n in ((q, "q"), (k, "k"), (v, "v"), (out, "out"))]
        ptrs = [_ints(t, n, seqs + d, dev) for t, n, d in ((q_offsets, "q_offsets", 1), (k_offsets, "k_offsets", 1),
                                                           (q_lens, "q_lens", 0), (k_lens, "k_lens", 0))]
        nq, hq, d = q.shape
        nk, hk = k.shape[:2]
        need = _workspace_bytes(code, seqs, nq, nk, hq, hk, d, left, right, sinks)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        s = _stream(q, stream, out, ws)
        _l.check(_l.load().nq_window_attention(
            *(ctypes.byref(r) for r in rows), code, seqs, nq, nk, *ptrs, hq, hk, d, left, right, sinks,
            d ** -0.5 if scale is None else scale, ws.data_ptr() if need else None, need, s))
    return out
