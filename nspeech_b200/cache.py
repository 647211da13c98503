"""A key / value cache in pages, with its bookkeeping on the device (``nq_cache_*``).

A slot holds one sequence: a row of page numbers and a length.  Slots share pages (``fork``), take copies of a shared
last page when they grow (``reserve``), give pages back (``free``, ``trim``), and ``compact`` brings the live pages
together.  Every call works on a range of slots ``[first, first + n)``, is a fixed number of launches without host
synchronisation, and can be captured into a CUDA graph.  It takes the place of the reference's ``kv_cache_append`` and
of its decoder's contiguous caches (src/moonshine/gpu_decoder.rs:21-88) for batches and beams.

A decoding step: ``reserve`` once, then per layer ``write`` and ``attention``.  A call that cannot be done (no free
pages, a full slot, a bad index) changes nothing, and the calls after it do nothing, until ``check`` has raised it.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import lib as _l
from .attention import _Pair, _code, _device, _ints, _output, _ref, _rows, _stream
from .fast_matmul import MatMulError


class PagedCache:
    """Pages k, v [layers, pages, kv_heads, page_tokens, head_dim] (f32 or bf16), table int32 [slots, max_pages] (-1: no
    page), lens int32 [slots], refs int32 [pages]: the caller's contiguous CUDA tensors, read and updated in place."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor):
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype:
            raise MatMulError("k and v must be [layers, pages, kv_heads, page_tokens, head_dim] of one dtype")
        code = _code(k, "k")
        if table.dim() != 2:
            raise MatMulError("table must be [slots, max_pages]")
        layers, pages, heads, tokens, dim = k.shape
        slots, max_pages = table.shape
        for t, name, shape in ((k, "k", k.shape), (v, "v", k.shape), (table, "table", table.shape), (lens, "lens", (slots,)),
                               (refs, "refs", (pages,))):
            if t.device != k.device or not t.is_contiguous() or tuple(t.shape) != tuple(shape):
                raise MatMulError(f"{name} must be contiguous {list(shape)} on {k.device}")
        for t, name in ((table, "table"), (lens, "lens"), (refs, "refs")):
            if t.dtype != torch.int32:
                raise MatMulError(f"{name} must be int32")
        self._dev = _device(k, "k")
        ints = _l.load().nq_cache_state_ints(slots, pages)
        if ints < 0:
            _l.check(int(ints))
        self.state = torch.zeros(ints, dtype=torch.int32, device=k.device)
        self.k, self.v, self.table, self.lens, self.refs = k, v, table, lens, refs
        self.device = k.device
        self._c = _l.Cache(k.data_ptr(), v.data_ptr(), table.data_ptr(), lens.data_ptr(), refs.data_ptr(), self.state.data_ptr(),
                           code, layers, pages, tokens, heads, dim, slots, max_pages)
        self._p = ctypes.byref(self._c)
        self._ws: dict = {}  # workspace sizes by call shape

    @classmethod
    def create(cls, layers: int, pages: int, page_tokens: int, kv_heads: int, head_dim: int, slots: int, max_pages: int,
               dtype: torch.dtype = torch.bfloat16, device=0) -> "PagedCache":
        """An empty cache of new tensors."""
        dev = torch.device("cuda", device) if isinstance(device, int) else torch.device(device)
        pool = [torch.zeros((layers, pages, kv_heads, page_tokens, head_dim), dtype=dtype, device=dev) for _ in range(2)]
        return cls(*pool, torch.full((slots, max_pages), -1, dtype=torch.int32, device=dev),
                   *(torch.zeros(n, dtype=torch.int32, device=dev) for n in (slots, pages)))

    @property
    def slots(self) -> int:
        return self._c.slots

    @property
    def live(self) -> torch.Tensor:
        """Live pages as of the last ``compact``: a CUDA int32 [1]."""
        return self.state[1:2]

    def _call(self, fn, *args) -> None:
        """A call with this cache's device as the current one."""
        if torch.cuda.current_device() == self._dev:
            rc = fn(self._p, *args)
        else:
            with torch.cuda.device(self._dev):
                rc = fn(self._p, *args)
        if rc:
            _l.check(rc)

    def _range(self, new, first: int, n: Optional[int]):
        """New tokens per slot: (offsets pointer, tokens each, slots)."""
        if isinstance(new, torch.Tensor):
            n = new.numel() - 1 if n is None else n
            return _ints(new, "offsets", n + 1, self._dev), 0, n
        return None, int(new), self.slots - first if n is None else n

    # ------------------------------------------------------------------ pages
    def reserve(self, tokens, first: int = 0, n: Optional[int] = None, stream: Optional[torch.cuda.Stream] = None) -> None:
        """Room for new tokens of slots [first, first + n): `tokens` each, or offsets [n + 1] (CUDA int32) whose
        differences are their numbers.  Takes the lowest free pages in slot order; a shared partial last page is copied."""
        off, each, n = self._range(tokens, first, n)
        self._call(_l.load().nq_cache_reserve, first, n, off, each, _stream(self._dev, stream))

    def write(self, k: torch.Tensor, v: torch.Tensor, tokens, first: int = 0, n: Optional[int] = None, layer: int = 0,
              stream: Optional[torch.cuda.Stream] = None) -> None:
        """The reserved tokens' keys and values, [rows, kv_heads, head_dim] for `layer` or [layers, rows, kv_heads,
        head_dim] for the layers from `layer` on; `tokens` as in ``reserve``."""
        off, each, n = self._range(tokens, first, n)
        shape, dtype = k.shape, self.k.dtype
        if shape != v.shape or len(shape) not in (3, 4) or shape[-2] != self._c.kv_heads or shape[-1] != self._c.head_dim:
            raise MatMulError(f"k and v must be [(layers,) rows, {self._c.kv_heads}, {self._c.head_dim}]")
        if len(shape) == 4:
            layers, by = shape[0], (k.stride(0), v.stride(0))
            if layers == 0:
                return
            k, v = k[0], v[0]
        else:
            layers, by = 1, (0, 0)
        rows = _Pair(_rows(k, "k", dtype, self._dev), _rows(v, "v", dtype, self._dev))
        self._call(_l.load().nq_cache_write, rows, _ref(rows, 24), *by, layer, layers, shape[-3], first, n, off, each,
                   _stream(self._dev, stream))

    def fork(self, src: torch.Tensor, first: int = 0, stream: Optional[torch.cuda.Stream] = None) -> None:
        """Slots [first, first + len(src)) become what slots `src` (CUDA int32) were before; -1 frees."""
        self._call(_l.load().nq_cache_fork, first, src.numel(), _ints(src, "src", None, self._dev), _stream(self._dev, stream))

    def free(self, first: int = 0, n: Optional[int] = None, stream: Optional[torch.cuda.Stream] = None) -> None:
        """Empties slots [first, first + n)."""
        self._call(_l.load().nq_cache_fork, first, self.slots - first if n is None else n, None, _stream(self._dev, stream))

    def trim(self, window: int, sinks: int = 0, first: int = 0, n: Optional[int] = None,
             stream: Optional[torch.cuda.Stream] = None) -> None:
        """Gives back pages that hold neither one of a slot's first `sinks` tokens nor one of its last `window`."""
        self._call(_l.load().nq_cache_trim, first, self.slots - first if n is None else n, sinks, window, _stream(self._dev, stream))

    def compact(self, stream: Optional[torch.cuda.Stream] = None) -> None:
        """Moves the live pages to the lowest numbers (``live`` of them); tables follow."""
        self._call(_l.load().nq_cache_compact, _stream(self._dev, stream))

    def check(self, stream: Optional[torch.cuda.Stream] = None) -> None:
        """Synchronises and raises NqError if a call since the last check could not be done."""
        self._call(_l.load().nq_cache_status, None, _stream(self._dev, stream))

    # -------------------------------------------------------------- attention
    def attention(self, q: torch.Tensor, layer: int, offsets: Optional[torch.Tensor] = None, first: int = 0,
                  n: Optional[int] = None, left: int = -1, right: int = 0, sinks: int = 0, scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """Attention of q [rows, q_heads, head_dim], the last tokens of slots [first, first + n) (offsets [n + 1], or the
        same number each), over their cached tokens; window and sinks as in ``window_attention``."""
        sq, dtype = q.shape, self.k.dtype
        if len(sq) != 3 or sq[2] != self._c.head_dim or sq[1] % self._c.kv_heads:
            raise MatMulError(f"q must be [rows, a multiple of {self._c.kv_heads} heads, {self._c.head_dim}]")
        if n is None:
            n = offsets.numel() - 1 if offsets is not None else self.slots - first
        out = _output(out, q)
        rows = _Pair(_rows(q, "q", dtype, self._dev), _rows(out, "out", dtype, self._dev))
        key = (n, sq[0], sq[1], left, right, sinks)
        need = self._ws.get(key)
        if need is None:
            need = _l.load().nq_cache_attention_workspace(self._p, *key)
            if need < 0:
                _l.check(int(need))
            if len(self._ws) > 4096:
                self._ws.clear()
            self._ws[key] = need
        ws = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
        self._call(_l.load().nq_cache_attention, layer, rows, _ref(rows, 24), first, n, sq[0],
                   _ints(offsets, "offsets", n + 1, self._dev), sq[1], left, right, sinks,
                   sq[2] ** -0.5 if scale is None else scale, ws.data_ptr() if need else None, need,
                   _stream(self._dev, stream, out, ws))
        return out
