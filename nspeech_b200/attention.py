"""Attention through a sliding window with sinks (``nq_window_attention``).

The reference's decoders and Moonshine's encoder run it between the matmuls
(``flash_attention_fwd``, kernels/moonshine_kernels.py:749-845; sliding window
of src/moonshine/encoder.rs:116-135).  Of a sequence with n_q queries and n_k
keys, query i stands at position ``p = n_k - n_q + i`` and sees key j when
``j <= p + right`` and (``j >= p - left`` or ``j < sinks``); a negative left or
right is no limit.  ``nspeech_b200.cache`` runs the same over a paged cache.
"""
from __future__ import annotations

import ctypes
import functools
from typing import Optional

import torch

from . import lib as _l
from .fast_matmul import MatMulError

_CODES = {torch.float32: _l.NQ_F32, torch.bfloat16: _l.NQ_BF16}
_ref = ctypes.byref
_Quad = _l.Rows * 4
_Pair = _l.Rows * 2


def _code(t: torch.Tensor, name: str) -> int:
    code = _CODES.get(t.dtype)
    if code is None:
        raise MatMulError(f"{name} has dtype {t.dtype} (f32 or bf16)")
    return code


def _device(t: torch.Tensor, name: str) -> int:
    """The tensor's device, made ready."""
    index = t.get_device()
    if index not in _l._inited:
        if not t.is_cuda:
            raise MatMulError(f"{name} must live on a CUDA device")
        now = torch.cuda.current_device()
        _l.init(index)
        torch.cuda.set_device(now)
    return index


def _stream(index: int, stream: Optional[torch.cuda.Stream], *made: Optional[torch.Tensor]) -> int:
    """The stream to launch on: `stream`, or the current one of the device.  Tensors made for the call on the current
    stream are kept from reuse until `stream` is through with them."""
    if stream is None:
        return torch.cuda.current_stream(index).cuda_stream
    if stream.device.index != index:
        raise MatMulError(f"the stream is on {stream.device}, the tensors on cuda:{index}")
    for m in made:
        if m is not None:
            m.record_stream(stream)
    return stream.cuda_stream


def _rows(t: torch.Tensor, name: str, dtype: torch.dtype, index: int):
    """(address, token stride, head stride) of rows [token][head][head_dim]."""
    st = t.stride()
    if t.dtype != dtype or t.get_device() != index or len(st) != 3 or (st[2] != 1 and t.shape[2] > 1 and t.numel()):
        raise MatMulError(f"{name} must be [rows, heads, head_dim] of {dtype} on cuda:{index} with unit last stride")
    return t.data_ptr(), st[0], st[1]


def _ints(t: Optional[torch.Tensor], name: str, n: Optional[int], index: int) -> Optional[int]:
    if t is None:
        return None
    if t.dtype != torch.int32 or t.dim() != 1 or t.get_device() != index or not t.is_contiguous() or (n is not None and t.numel() != n):
        raise MatMulError(f"{name} must be contiguous int32{'' if n is None else f' [{n}]'} on cuda:{index}")
    return t.data_ptr()


def _output(out: Optional[torch.Tensor], q: torch.Tensor) -> torch.Tensor:
    if out is None:
        return torch.empty_like(q, memory_format=torch.contiguous_format)
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
    sq, sk = q.shape, k.shape
    if len(sq) != 3 or len(sk) != 3:
        raise MatMulError("q, k and v must be [rows, heads, head_dim]")
    nq, hq, d = sq
    nk, hk, dk = sk
    if v.shape != sk or dk != d or hk == 0 or hq % hk:
        raise MatMulError(f"q {tuple(sq)}, k {tuple(sk)} and v {tuple(v.shape)} do not fit together")
    dtype = q.dtype
    code, dev = _code(q, "q"), _device(q, "q")
    if dev != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return window_attention(q, k, v, left, right, sinks, scale, q_offsets, k_offsets, q_lens, k_lens, seqs, out, stream)
    if seqs is None:
        seqs = (q_offsets.numel() - 1 if q_offsets is not None else k_offsets.numel() - 1 if k_offsets is not None else
                q_lens.numel() if q_lens is not None else k_lens.numel() if k_lens is not None else 1)
    out = _output(out, q)
    rows = _Quad(_rows(q, "q", dtype, dev), _rows(k, "k", dtype, dev), _rows(v, "v", dtype, dev), _rows(out, "out", dtype, dev))
    need = _workspace_bytes(code, seqs, nq, nk, hq, hk, d, left, right, sinks)
    ws = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    rc = _l.load().nq_window_attention(
        rows, _ref(rows, 24), _ref(rows, 48), _ref(rows, 72), code, seqs, nq, nk, _ints(q_offsets, "q_offsets", seqs + 1, dev),
        _ints(k_offsets, "k_offsets", seqs + 1, dev), _ints(q_lens, "q_lens", seqs, dev), _ints(k_lens, "k_lens", seqs, dev),
        hq, hk, d, left, right, sinks, d ** -0.5 if scale is None else scale, ws.data_ptr() if need else None, need,
        _stream(dev, stream, out, ws))
    if rc:
        _l.check(rc)
    return out
