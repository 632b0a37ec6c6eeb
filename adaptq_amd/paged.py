"""``PagedCache``: exact keys and values in pages that sequences share, and ``PagedCache4``,
the same in 4 bits (adaptq_paged_* and adaptq_paged4_* of adaptq.h).

    cache = PagedCache.allocate(pages, heads=8, page_size=64, dim=128, rotary=Rotary(128))
    cache.append(k, v, table, lengths, offsets)   # prompts: rotated keys and values into pages
    out = cache.step(q, k, v, table, lengths)     # one token a sequence: append, then attend
    lengths += 1                                  # the caller keeps tables and lengths

Sequence b's token p lies in page ``table[b, p // page_size]``, slot ``p % page_size``;
``lengths[b]`` is what it holds before the call.  All tensors are on the GPU, the table,
lengths and offsets int32; calls run on torch's current stream, allocate only their
output (and, where prompts are short or weights are asked for, a workspace), never wait, and
may be captured into a graph, which the cache has to outlive.
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


class _Pages:
    """What caches in pages share: their geometry, the order of calls, checks of arguments."""

    def _start(self, k_pages, v_pages, dim, dtype, rotary, kind):
        self._io = IO_TYPES[dtype]
        if not k_pages.is_contiguous() or not v_pages.is_contiguous():
            raise ValueError("pages must be contiguous")
        self.device = k_pages.device
        if self.device.type != "cuda" or v_pages.device != self.device:
            raise ValueError("pages must be on one GPU")
        if rotary is not None and rotary.device != self.device:
            raise ValueError(f"the rotary is on {rotary.device}, the pages on {self.device}")
        self.k_pages, self.v_pages = self._pools = k_pages, v_pages
        self.pages, self.heads, self.page_size = k_pages.shape[:3]
        self.dim, self.dtype = dim, dtype
        self._size = torch.finfo(dtype).bits // 8
        self._last = None  # the stream of the last call, and its address
        self._last_address = None
        with torch.cuda.device(self.device):
            self._handle = kind(k_pages.data_ptr(), v_pages.data_ptr(), self.pages,
                                self.page_size, self.heads, dim, self._io,
                                None if rotary is None else rotary._handle)

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
            offsets = self._offsets(offsets, lengths)
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

    def _step_rows(self, k, v, lengths):
        """A step's rows as the library takes them, and the tensors that hold them."""
        k, v = self._rows(k, "k", self.heads), self._rows(v, "v", self.heads)
        if k.shape[0] != lengths.shape[0] or v.shape[0] != k.shape[0]:
            raise ValueError("k and v hold one token a sequence")
        size, ks, vs = self._size, k.stride(), v.stride()
        return (k.data_ptr(), v.data_ptr(), ks[1] * size, ks[0] * size, vs[1] * size,
                vs[0] * size), k, v

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

    def _offsets(self, offsets, lengths):
        if offsets.dtype != torch.int32 or offsets.shape != (lengths.shape[0] + 1,):
            raise ValueError("offsets must be int32 [sequences + 1]")
        if offsets.device != self.device:
            raise ValueError(f"offsets must be on {self.device}")
        return offsets.contiguous()

    def _scores(self, n, q_heads, softcap, slopes, prefix, first):
        """What attention with scores of its own takes: (softcap, slopes, prefix, first)."""
        if softcap is not None and not softcap >= 2.0 ** -100:  # 0 in fp32 would mean none
            raise ValueError(f"softcap must be positive, 2^-100 or more, got {softcap}")
        at = []
        for name, x, dtype, size in (("slopes", slopes, torch.float32, q_heads),
                                     ("prefix", prefix, torch.int32, n),
                                     ("first", first, torch.int32, n)):
            if x is None:
                at.append(0)
                continue
            if x.dtype != dtype or x.shape != (size,):
                raise ValueError(f"{name} must be {dtype} [{size}], got {x.dtype} "
                                 f"{tuple(x.shape)}")
            if x.device != self.device:
                raise ValueError(f"{name} must be on {self.device}")
            if size > 1 and x.stride(0) != 1:
                raise ValueError(f"{name} must lie side by side")
            at.append(x.data_ptr())
        return (softcap or 0.0, *at)

    def _queries(self, q, lengths, scale, window, out):
        q = self._rows(q, "q", 0)
        if lengths is not None and q.shape[0] != lengths.shape[0]:
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


class PagedCache(_Pages):
    """A cache over two tensors [pages, heads, page_size, dim] of fp32, fp16 or bf16:
    page_size a multiple of 16, dim a multiple of 8 up to 256.  With ``rotary``, appended
    keys and the queries of attention are rotated by their positions."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 rotary: Rotary | None = None):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape:
            raise ValueError("k_pages and v_pages must be [pages, heads, page_size, dim], got "
                             f"{tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
        if k_pages.dtype not in IO_TYPES or v_pages.dtype != k_pages.dtype:
            raise TypeError("pages must be float32, float16 or bfloat16, both alike")
        self._start(k_pages, v_pages, k_pages.shape[3], k_pages.dtype, rotary,
                    adaptq_py.PagedCache)
        self._rotates = rotary is not None

    @classmethod
    def allocate(cls, pages: int, heads: int, page_size: int, dim: int,
                 dtype: torch.dtype = torch.bfloat16, device=None,
                 rotary: Rotary | None = None) -> "PagedCache":
        """A cache over new pools (their contents undefined until appended to)."""
        device = torch.device("cuda" if device is None else device)
        k, v = (torch.empty(pages, heads, page_size, dim, dtype=dtype, device=device)
                for _ in range(2))
        return cls(k, v, rotary)

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
               offsets: torch.Tensor | None = None, *, scale: float | None = None,
               window: int | None = None, softcap: float | None = None,
               slopes: torch.Tensor | None = None, prefix: torch.Tensor | None = None,
               first: torch.Tensor | None = None, weights: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Attention of one query a sequence, q [sequences, q_heads, dim], over its tokens
        (the last ``window`` of them); q_heads a multiple of heads.  q is the token at
        lengths - 1.  scale: 1/sqrt(dim).  Sequences without tokens give zeros.

        With offsets, of several: q [tokens, q_heads, dim], tokens offsets[b] to
        offsets[b + 1] - 1 the last ones of sequence b, whose lengths[b] counts them (a prompt
        after its append); rows outside the offsets are left as ``out`` has them (without it
        they hold anything).

        For the query at position p and token t: scores become softcap * tanh(score / softcap),
        then lose slopes[q_head] * |p - t| (float32); t is seen where first <= t and
        (t < prefix or p - window < t <= p).  prefix and first are int32, one a query.

        weights, float32 [sequences, heads, table's columns * page_size or more], of one query a
        sequence: to each token that is seen, the sum of its weights over the query heads of a
        key head is added."""
        seqs = self._sequences(table, lengths)
        if offsets is not None:
            if weights is not None:
                raise ValueError("weights are added up of one query a sequence, without offsets")
            offsets = self._offsets(offsets, lengths)
            q, y, args = self._queries(q, None, scale, window, out)
            n = q.shape[0]
            if n and seqs[4]:
                shape = self._scores(n, q.shape[1], softcap, slopes, prefix, first)
                need = self._handle.prompt_workspace(q.shape[1], n, seqs[4], seqs[1], args[1][1],
                                                     *shape[2:])
                space = torch.empty(need, dtype=torch.uint8, device=self.device) if need else None
                self._handle.prompt(*args[0], n, *seqs, offsets.data_ptr(), *args[1], *shape,
                                    0 if space is None else space.data_ptr(), need,
                                    self._stream())
                if out is not None:
                    increment_version((out,))
            return y
        q, y, args = self._queries(q, lengths, scale, window, out)
        if q.shape[0]:
            if softcap is slopes is prefix is first is weights is None:
                self._handle.attend(*args[0], *seqs, *args[1], self._stream())
            else:
                self._scored((0,) * 6, args, seqs, softcap, slopes, prefix, first, weights)
            if out is not None:
                increment_version((out,))
        return y

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
             lengths: torch.Tensor, *, scale: float | None = None, window: int | None = None,
             softcap: float | None = None, slopes: torch.Tensor | None = None,
             prefix: torch.Tensor | None = None, first: torch.Tensor | None = None,
             weights: torch.Tensor | None = None,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """append(k, v) with one token a sequence, then attend(q) over lengths + 1."""
        seqs = self._sequences(table, lengths)
        rows = self._step_rows(k, v, lengths)
        q, y, args = self._queries(q, lengths, scale, window, out)
        if q.shape[0]:
            if softcap is slopes is prefix is first is weights is None:
                self._handle.step(*rows[0], *args[0], *seqs, *args[1], self._stream())
            else:
                self._scored(rows[0], args, seqs, softcap, slopes, prefix, first, weights)
            increment_version(self._pools if out is None else (*self._pools, out))
        return y

    def evict(self, weights: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
              keep: int, *, recent: int = 0, into: torch.Tensor | None = None) -> torch.Tensor:
        """Of each sequence and key head that holds more, ``keep`` tokens stay: the ``recent``
        last ones, and of the others those of the largest weights (of equal ones the earlier).
        They move, in their order, to the sequence's first places, their weights too (with
        zeros behind), so that after it

            kept = cache.evict(weights, table, lengths, keep)
            lengths.clamp_(max=keep)

        weights as attend adds them up.  into, int32 [sequences, pages for keep tokens]: other
        pages to move to, with nothing of the sequences in them (sequences of up to keep tokens
        are copied whole); without it a page may be no second sequence's.  Returns where the
        tokens lay, int32 [sequences, heads, keep], -1 where there are none.  Refused where the
        cache rotates: positions come from lengths then.  Later calls' slopes, window, first and
        prefix count the places that are left, not the tokens that were there."""
        seqs = self._sequences(table, lengths)
        if self._rotates:
            raise ValueError("a cache with a rotary takes positions from its lengths, which "
                             "eviction changes: rotate rows before they are appended")
        if not 0 < keep < 2 ** 31 or not 0 <= recent <= keep:
            raise ValueError(f"keep must be positive, recent from 0 to keep, got {keep}, {recent}")
        w = self._weights(weights, seqs)
        where = (0, 0, 0)
        if into is not None:
            n = lengths.shape[0]
            if into.dtype != torch.int32 or into.dim() != 2 or into.shape[0] != n or \
                    into.shape[1] * self.page_size < keep:
                raise ValueError("into must be int32 [sequences, pages for keep tokens], got "
                                 f"{into.dtype} {tuple(into.shape)}")
            if into.device != self.device:
                raise ValueError(f"into must be on {self.device}")
            into = into.contiguous()
            where = into.data_ptr(), into.shape[1], into.shape[1]
        kept = torch.empty(seqs[4], self.heads, keep, dtype=torch.int32, device=self.device)
        if seqs[4]:
            self._handle.evict(*w, *seqs, keep, recent, *where, kept.data_ptr(), self._stream())
            increment_version((*self._pools, weights))
        return kept

    def _scored(self, rows, args, seqs, softcap, slopes, prefix, first, weights):
        shape = self._scores(seqs[4], args[0][2], softcap, slopes, prefix, first)
        w, space, need = (0, 0, 0), None, 0
        if weights is not None:
            w = self._weights(weights, seqs)
            need = self._handle.weights_workspace(args[0][2], seqs[4], seqs[1])
            space = torch.empty(need, dtype=torch.uint8, device=self.device)
        self._handle.scored(*rows, *args[0], *seqs, *args[1], *shape, *w,
                            0 if space is None else space.data_ptr(), need, self._stream())
        if weights is not None:
            increment_version((weights,))

    def _weights(self, weights, seqs):
        n, tokens = seqs[4], seqs[1] * self.page_size
        if weights.dtype != torch.float32 or weights.dim() != 3 or \
                weights.shape[:2] != (n, self.heads) or weights.shape[2] < tokens:
            raise ValueError(f"weights must be float32 [{n}, {self.heads}, {tokens} or more], got "
                             f"{weights.dtype} {tuple(weights.shape)}")
        if weights.device != self.device:
            raise ValueError(f"weights must be on {self.device}")
        s = weights.stride()
        if tokens > 1 and s[2] != 1:
            raise ValueError("a token's weights must lie side by side")
        return weights.data_ptr(), 4 * s[1], 4 * s[0]


class PagedCache4(_Pages):
    """A cache of 4-bit values: pools uint8 [pages, heads, page_size, 17 * dim / 32], page_size a
    multiple of 16, dim a multiple of 32 up to 256; what lies in them is the library's.  Rows
    go in and queries come in ``dtype``.

    32 channels of a row share a power of two, the smallest that takes the largest of them to 6
    or below; a value is held as its sign and the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (of two
    the even code), 32 with an infinity or NaN among them as NaN.  append, attend and step are
    PagedCache's, attention over the values as they are held."""

    def __init__(self, k_pages: torch.Tensor, v_pages: torch.Tensor, *,
                 dtype: torch.dtype = torch.bfloat16, rotary: Rotary | None = None):
        if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.shape[3] % 17:
            raise ValueError("k_pages and v_pages must be [pages, heads, page_size, 17 * dim / 32]"
                             f", got {tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
        if k_pages.dtype != torch.uint8 or v_pages.dtype != torch.uint8:
            raise TypeError("pages of 4-bit values must be uint8")
        if dtype not in IO_TYPES:
            raise TypeError(f"rows must be float32, float16 or bfloat16, got {dtype}")
        self._start(k_pages, v_pages, k_pages.shape[3] // 17 * 32, dtype, rotary,
                    adaptq_py.PagedCache4)

    @classmethod
    def allocate(cls, pages: int, heads: int, page_size: int, dim: int,
                 dtype: torch.dtype = torch.bfloat16, device=None,
                 rotary: Rotary | None = None) -> "PagedCache4":
        """A cache over new pools (their contents undefined until appended to)."""
        if dim <= 0 or dim % 32:
            raise ValueError(f"dim must be a multiple of 32, got {dim}")
        device = torch.device("cuda" if device is None else device)
        k, v = (torch.empty(pages, heads, page_size, dim // 32 * 17, dtype=torch.uint8,
                            device=device) for _ in range(2))
        return cls(k, v, dtype=dtype, rotary=rotary)

    def read(self, tokens: int, table: torch.Tensor, lengths: torch.Tensor,
             offsets: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
        """The keys and values, float32 [tokens, heads, dim], of the tokens that an append of
        as many with these arguments writes; zeros where there is no page."""
        seqs = self._sequences(table, lengths)
        at = 0
        if offsets is not None:
            offsets = self._offsets(offsets, lengths)
            at = offsets.data_ptr()
        elif tokens != lengths.shape[0]:
            raise ValueError("without offsets, one token a sequence is read")
        k, v = (torch.empty(tokens, self.heads, self.dim, dtype=torch.float32, device=self.device)
                for _ in range(2))
        if tokens and not seqs[4]:
            return k.zero_(), v.zero_()
        if tokens:
            self._handle.read(k.data_ptr(), v.data_ptr(), tokens, *seqs, at, self._stream())
        return k, v

    def attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *,
               scale: float | None = None, window: int | None = None,
               softcap: float | None = None, slopes: torch.Tensor | None = None,
               prefix: torch.Tensor | None = None, first: torch.Tensor | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """PagedCache.attend of one query a sequence, over the values as they are held."""
        seqs = self._sequences(table, lengths)
        q, y, args = self._queries(q, lengths, scale, window, out)
        if q.shape[0]:
            shape = self._scores(q.shape[0], q.shape[1], softcap, slopes, prefix, first)
            self._handle.scored(0, 0, 0, 0, 0, 0, *args[0], *seqs, *args[1], *shape,
                                self._stream())
            if out is not None:
                increment_version((out,))
        return y

    def step(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor,
             lengths: torch.Tensor, *, scale: float | None = None, window: int | None = None,
             softcap: float | None = None, slopes: torch.Tensor | None = None,
             prefix: torch.Tensor | None = None, first: torch.Tensor | None = None,
             out: torch.Tensor | None = None) -> torch.Tensor:
        """append(k, v) with one token a sequence, then attend(q) over lengths + 1."""
        seqs = self._sequences(table, lengths)
        rows = self._step_rows(k, v, lengths)
        q, y, args = self._queries(q, lengths, scale, window, out)
        if q.shape[0]:
            shape = self._scores(q.shape[0], q.shape[1], softcap, slopes, prefix, first)
            self._handle.scored(*rows[0], *args[0], *seqs, *args[1], *shape, self._stream())
            increment_version(self._pools if out is None else (*self._pools, out))
        return y
