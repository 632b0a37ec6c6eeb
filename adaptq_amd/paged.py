"""``PagedCache``: exact keys and values in pages that sequences share
(adaptq_paged_* of adaptq.h).

    cache = PagedCache.allocate(pages, heads=8, page_size=64, dim=128, rotary=Rotary(128))
    cache.append(k, v, table, lengths, offsets)   # prompts: rotated keys and values into pages
    out = cache.step(q, k, v, table, lengths)     # one token a sequence: append, then attend
    lengths += 1                                  # the caller keeps tables and lengths

Sequence b's token p lies in page ``table[b, p // page_size]``, slot ``p % page_size``;
``lengths[b]`` is what it holds before the call.  All tensors are on the GPU, the table,
lengths and offsets int32; calls run on torch's current stream, allocate only their
output, never wait, and may be captured into a graph, which the cache has to outlive.
Inference only: no gradients, and tracing (torch.jit.trace, make_fx, torch.export) is
refused.
Calls on one cache from different streams wait for each other (they share its workspace as
well as its pages; a stream that torch does not own has to outlive the cache's next call).
Replays of a graph are ordered by the caller, among each other and with calls: those that run
over each other give wrong outputs, and may leave the workspace such that later ones do.
"""
from __future__ import annotations

import torch

from . import adaptq_py
from .rotary import (IO_TYPES, Rotary, dispatch_modes, increment_version, refuse_tracing,
                     stream_of, tracing_state)


class PagedCache:
    """A cache over two tensors [pages, heads, page_size, dim] of fp32, fp16 or bf16:
    page_size a multiple of 16, dim a multiple of 8 up to 256.  With ``rotary``, appended
    keys and the queries of attention are rotated by their positions."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 rotary: Rotary | None = None):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
            raise ValueError("k_pages and v_pages must be [pages, heads, page_size, dim], got "
                             f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
        self._io = IO_TYPES.get(k_pages.dtype)
        if self._io is None or v_pages.dtype != k_pages.dtype:
            raise TypeError("pages must be float32, float16 or bfloat16, both alike")
        if not k_pages.is_contiguous() or not v_pages.is_contiguous():
            raise ValueError("pages must be contiguous")
        self.device = k_pages.device
        if self.device.type != "cuda" or v_pages.device != self.device:
            raise ValueError("pages must be on one GPU")
        if rotary is not None and rotary.device != self.device:
            raise ValueError(f"the rotary is on {rotary.device}, the pages on {self.device}")
        self.k_pages, self.v_pages = self._pools = k_pages, v_pages
        self.pages, self.heads, self.page_size, self.dim = k_pages.shape
        self.dtype = k_pages.dtype
        self._size = k_pages.element_size()
        self._last = None  # the stream of the last call, and its address
        self._last_address = None
        with torch.cuda.device(self.device):
            self._handle = adaptq_py.PagedCache(k_pages.data_ptr(), v_pages.data_ptr(), self.pages,
                                                self.page_size, self.heads, self.dim, self._io,
                                                None if rotary is None else rotary._handle)

    @classmethod
    def allocate(cls, pages: int, heads: int, page_size: int, dim: int,
                 dtype: torch.dtype = torch.bfloat16, device=None,
                 rotary: Rotary | None = None) -> "PagedCache":
        """A cache over new pools (their contents undefined until appended to)."""
        device = torch.device("cuda" if device is None else device)
        k, v = (torch.empty(pages, heads, page_size, dim, dtype=dtype, device=device)
                for _ in range(2))
        return cls(k, v, rotary)

    def append(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
               lengths: torch.Tensor, offsets: torch.Tensor | None = None) -> None:
        """Writes k, v [tokens, heads, dim]: tokens offsets[b] to offsets[b + 1] - 1 behind
        sequence b's lengths[b]; without offsets, token b of sequence b.  Tokens outside the
        offsets and positions without a page are left out."""
        seqs = self._sequences(table, lengths)
        k, v = self._rows(k, "k", self.heads), self._rows(v, "v", self.heads)
        if k.shape[0] != v.shape[0]:
            raise ValueError("k and v differ in tokens")
        at = 0
        if offsets is not None:
            if offsets.dtype != torch.int32 or offsets.shape != (lengths.shape[0] + 1,):
                raise ValueError("offsets must be int32 [sequences + 1]")
            if offsets.device != self.device:
                raise ValueError(f"offsets must be on {self.device}")
            offsets = offsets.contiguous()
            at = offsets.data_ptr()
        elif k.shape[0] != lengths.shape[0]:
            raise ValueError("without offsets, k and v hold one token a sequence")
        size, ks, vs = self._size, k.stride(), v.stride()
        if not k.shape[0]:
            return
        self._handle.append(k.data_ptr(), v.data_ptr(), k.shape[0], ks[1] * size, ks[0] * size,
                            vs[1] * size, vs[0] * size, *seqs, at, self._stream())
        # a graph that saved the pools sees that they changed, as torch's own writes do
        increment_version(self._pools)

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
               scale: float | None = None, window: int | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of one query a sequence, q [sequences, q_heads, dim], over its tokens
        (the last ``window`` of them); q_heads a multiple of heads.  q is the token at
        lengths - 1.  scale: 1/sqrt(dim).  Sequences without tokens give zeros."""
        seqs = self._sequences(table, lengths)
        q, y, args = self._queries(q, lengths, scale, window, out)
        if q.shape[0]:
            self._handle.attend(*args[0], *seqs, *args[1], self._stream())
            if out is not None:
                increment_version((out,))
        return y

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
             lengths: torch.Tensor, *, scale: float | None = None, window: int | None = None,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """append(k, v) with one token a sequence, then attend(q) over lengths + 1."""
        seqs = self._sequences(table, lengths)
        k, v = self._rows(k, "k", self.heads), self._rows(v, "v", self.heads)
        if k.shape[0] != lengths.shape[0] or v.shape[0] != k.shape[0]:
            raise ValueError("k and v hold one token a sequence")
        q, y, args = self._queries(q, lengths, scale, window, out)
        if q.shape[0]:
            size, ks, vs = self._size, k.stride(), v.stride()
            self._handle.step(k.data_ptr(), v.data_ptr(), ks[1] * size, ks[0] * size,
                              vs[1] * size, vs[0] * size, *args[0], *seqs, *args[1],
                              self._stream())
            increment_version(self._pools if out is None else (*self._pools, out))
        return y

    def _stream(self):
        address = stream_of(self.device)
        if address != self._last_address:
            self._follow(address)
        return address

    def _follow(self, address):
        """The current stream, which is not the last call's, waits for that one's work."""
        with torch.cuda.device(self.device):
            if torch.cuda.is_current_stream_capturing():
                return  # a capture waits for nothing outside it
            stream = torch.cuda.current_stream()
            if self._last is not None:
                with torch.cuda.stream(self._last):
                    captured = torch.cuda.is_current_stream_capturing()
                if not captured:  # (what waits for a captured stream is captured with it)
                    stream.wait_stream(self._last)
            self._last, self._last_address = stream, address

    def _rows(self, x, name, heads):
        if x.dim() != 3 or x.shape[2] != self.dim or heads and x.shape[1] != heads:
            raise ValueError(f"{name} must be [n, {heads or 'q_heads'}, {self.dim}], got "
                             f"{tuple(x.shape)}")
        if x.dtype != self.dtype:
            raise TypeError(f"{name} must be {self.dtype} as the pages, got {x.dtype}")
        if x.device != self.device:
            raise ValueError(f"{name} must be on {self.device}")
        return x if x.stride(2) == 1 else x.contiguous()

    def _sequences(self, table, lengths):
        if tracing_state() is not None or dispatch_modes():
            refuse_tracing("PagedCache")
        if table.dtype != torch.int32 or lengths.dtype != torch.int32:
            raise TypeError("table and lengths must be int32")
        n = lengths.shape[0] if lengths.dim() == 1 else -1
        if table.dim() != 2 or table.shape[0] != n:
            raise ValueError("table must be [sequences, width] and lengths [sequences], got "
                             f"{tuple(table.shape)} and {tuple(lengths.shape)}")
        if table.device != self.device or lengths.device != self.device:
            raise ValueError(f"table and lengths must be on {self.device}")
        width, stride = table.shape[1], table.stride(0)
        if width > 1 and table.stride(1) != 1 or n > 1 and stride < width or \
                n > 1 and lengths.stride(0) != 1:
            raise ValueError("table rows and lengths must lie side by side")
        return table.data_ptr(), width, max(stride, width), lengths.data_ptr(), n

    def _queries(self, q, lengths, scale, window, out):
        q = self._rows(q, "q", 0)
        if q.shape[0] != lengths.shape[0]:
            raise ValueError("q holds one query a sequence")
        if window is not None and window <= 0:
            raise ValueError(f"window must be positive, got {window}")
        if scale is not None and abs(scale) < 2.0 ** -126:  # 0 in fp32 would mean 1/sqrt(dim)
            raise ValueError(f"scale must not be 0 in fp32, got {scale}")
        if out is None:
            out = torch.empty_like(q)  # its rows' values side by side, as q's are
            if out.stride(2) != 1:  # (not where q's rows overlap)
                out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        elif self._rows(out, "out", 0) is not out or out.shape != q.shape:
            raise ValueError("out must have q's shape, its rows' values side by side")
        size, qs, os = self._size, q.stride(), out.stride()
        return q, out, ((q.data_ptr(), out.data_ptr(), q.shape[1], qs[1] * size, qs[0] * size,
                         os[1] * size, os[0] * size), (scale or 0.0, window or 0))
