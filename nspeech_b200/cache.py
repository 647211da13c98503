"""A key / value cache in pages, with its bookkeeping on the device (``nq_cache_*``).

A slot holds one sequence: a row of page numbers and a length.  Slots share pages (``fork``), take copies of a shared
last page when they grow (``reserve``), give pages back (``free``, ``trim``), and ``compact`` brings the live pages
together.  Every call works on a range of slots ``[first, first + n)``, is a fixed number of launches without host
synchronisation, and can be captured into a CUDA graph.  It takes the place of the reference's ``kv_cache_append`` and
of its decoder's contiguous caches (src/moonshine/gpu_decoder.rs:21-88) for batches and beams.

A decoding step: ``reserve`` once, then per layer ``write`` and ``attention``.  A call that cannot be done (no free
pages, a full slot, a bad index) changes nothing, and the calls that change the cache do nothing after it, until
``check`` has raised it; attention goes on over what is there.

Attention splits its keys by what a slot may hold, ``max_pages * page_tokens``, so take `max_pages` for the longest
sequence that there will be, not for more.
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import lib as _l
from .attention import _on
from .fast_matmul import MatMulError

_n = _l.native()


class PagedCache:
    """Pages k, v [layers, pages, kv_heads, page_tokens, head_dim] (f32 or bf16), table int32 [slots, max_pages] (-1: no
    page), lens int32 [slots], refs int32 [pages]: the caller's contiguous CUDA tensors, read and updated in place (autograd
    does not see it)."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, refs: torch.Tensor):
        if k.dim() != 5 or k.shape != v.shape or k.dtype != v.dtype:
            raise MatMulError("k and v must be [layers, pages, kv_heads, page_tokens, head_dim] of one dtype")
        if k.dtype not in (torch.float32, torch.bfloat16):
            raise MatMulError(f"the pages have dtype {k.dtype} (f32 or bf16)")
        if not k.is_cuda:
            raise MatMulError("the pages must live on a CUDA device")
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
        ints = _l.load().nq_cache_state_ints(slots, pages)
        if ints < 0:
            _l.check(int(ints))
        self.state = torch.zeros(ints, dtype=torch.int32, device=k.device)
        self.k, self.v, self.table, self.lens, self.refs = k, v, table, lens, refs
        self._c = _l.Cache(k.data_ptr(), v.data_ptr(), table.data_ptr(), lens.data_ptr(), refs.data_ptr(), self.state.data_ptr(),
                           _l.NQ_F32 if k.dtype == torch.float32 else _l.NQ_BF16, layers, pages, tokens, heads, dim, slots, max_pages)
        self._at = ctypes.addressof(self._c), k.device.index

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

    def _run(self, fn, args, stream: Optional[torch.cuda.Stream]):
        if stream is None:
            return fn(*self._at, *args)
        with _on(stream, self.k):
            return fn(*self._at, *args)

    # ------------------------------------------------------------------ pages
    def reserve(self, tokens, first: int = 0, n: Optional[int] = None, stream: Optional[torch.cuda.Stream] = None) -> None:
        """Room for new tokens of slots [first, first + n): `tokens` each, or offsets [n + 1] (CUDA int32) whose
        differences are their numbers.  Takes the lowest free pages in slot order; a shared partial last page is copied."""
        self._run(_n.cache_reserve, (tokens, first, n), stream)

    def write(self, k: torch.Tensor, v: torch.Tensor, tokens, first: int = 0, n: Optional[int] = None, layer: int = 0,
              stream: Optional[torch.cuda.Stream] = None) -> None:
        """The reserved tokens' keys and values, [rows, kv_heads, head_dim] for `layer` or [layers, rows, kv_heads,
        head_dim] for the layers from `layer` on; `tokens` as in ``reserve``."""
        self._run(_n.cache_write, (k, v, tokens, first, n, layer), stream)

    def fork(self, src: torch.Tensor, first: int = 0, stream: Optional[torch.cuda.Stream] = None) -> None:
        """Slots [first, first + len(src)) become what slots `src` (CUDA int32) were before; -1 frees."""
        if src is None:
            raise MatMulError("src must be a tensor")
        self._run(_n.cache_fork, (src, first, None), stream)

    def free(self, first: int = 0, n: Optional[int] = None, stream: Optional[torch.cuda.Stream] = None) -> None:
        """Empties slots [first, first + n)."""
        self._run(_n.cache_fork, (None, first, n), stream)

    def trim(self, window: int, sinks: int = 0, first: int = 0, n: Optional[int] = None,
             stream: Optional[torch.cuda.Stream] = None) -> None:
        """Gives back pages that hold neither one of a slot's first `sinks` tokens nor one of its last `window`."""
        self._run(_n.cache_trim, (window, sinks, first, n), stream)

    def compact(self, stream: Optional[torch.cuda.Stream] = None) -> None:
        """Moves the live pages to the lowest numbers (``live`` of them); tables follow."""
        self._run(_n.cache_compact, (), stream)

    def check(self, stream: Optional[torch.cuda.Stream] = None) -> None:
        """Synchronises and raises NqError if a call since the last check could not be done."""
        self._run(_n.cache_check, (), stream)

    # -------------------------------------------------------------- attention
    def attention(self, q: torch.Tensor, layer: int, offsets: Optional[torch.Tensor] = None, first: int = 0,
                  n: Optional[int] = None, left: int = -1, right: int = 0, sinks: int = 0, scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None, stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
        """Attention of q [rows, q_heads, head_dim], the last tokens of slots [first, first + n) (offsets [n + 1], or the
        same number each), over their cached tokens; window and sinks as in ``window_attention``."""
        return self._run(_n.cache_attention, (q, layer, offsets, first, n, left, right, sinks, scale, out), stream)
