"""A paged cache of keys and values for a batch that is being decoded.

The reference's attention modules keep past keys and values by concatenation
(trinix/layers/attention/grouped_query_attention.py:178-184): every step copies the whole cache. Here it is a pool of
pages of fixed size, in the activation's 16 bits or in 4 bits (`ops.append_paged`), of which each sequence of the
batch owns some; FastGroupedQueryAttention and FastMultiQueryAttention take one as `past_key_value`.
"""
from __future__ import annotations

from typing import List, Optional, Sequence, Tuple, Union

import torch

from . import ops


class PagedKVCache:
    """`num_pages` pages of `page_size` tokens for `num_kv_heads` heads of `head_dim`, shared by `batch_size`
    sequences of up to `max_pages` pages each (default: all of them; attention modules with rotation keep tables of so
    many positions).

    Which page is whose is kept on the host, with the lengths that the host has reserved room for; the block table
    and the lengths that the kernels read are on the device, so that a step (`reserve` aside) may be captured in a
    CUDA graph and replayed: reserve the steps' tokens first. What replays append the host does not see: from the
    first capture on, `reserve` and an `append` that is not captured read the lengths from the device before they
    look for room. A place of the batch without pages takes no tokens: its length stays 0, nothing of it is written,
    and its queries get 0. bits=4 holds each row of head_dim values in head_dim / 2 + 8 bytes.
    """

    def __init__(self, num_pages: int, page_size: int, num_kv_heads: int, head_dim: int, batch_size: int = 1, *,
                 max_pages: Optional[int] = None, bits: int = 16, dtype: torch.dtype = torch.bfloat16,
                 device: Union[str, torch.device] = "cuda"):
        if bits not in (4, 16):
            raise ValueError(f"a cache holds 16 or 4 bits, got {bits}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise TypeError("the paged cache serves bfloat16 and float16")
        if min(num_pages, num_kv_heads, batch_size) < 1 or page_size < 1 or page_size % 16 or page_size > 4096:
            raise ValueError("pages, heads and sequences must be positive, page_size a multiple of 16 up to 4096")
        if head_dim not in (64, 128):
            raise ValueError(f"the paged cache serves head_dim 64 and 128, got {head_dim}")
        self.page_size, self.bits, self.dtype = page_size, bits, dtype
        shape = (num_pages, num_kv_heads, page_size, head_dim if bits == 16 else head_dim // 2)
        held = dtype if bits == 16 else torch.uint8
        self.k_pages, self.v_pages = (torch.zeros(shape, dtype=held, device=device) for _ in range(2))
        self.k_scales = self.v_scales = None
        if bits == 4:
            self.k_scales, self.v_scales = (torch.zeros((*shape[:3], 2), dtype=torch.float32, device=device)
                                            for _ in range(2))
        self.max_pages = num_pages if max_pages is None else max_pages
        # a place's row: whether it has pages, then which
        self._table = torch.full((batch_size, 1 + self.max_pages), -1, dtype=torch.int32, device=device)
        self._table[:, 0] = 0
        self._in_use, self.block_table = self._table[:, 0], self._table[:, 1:]
        self.lengths = torch.zeros(batch_size, dtype=torch.int32, device=device)
        self._free: List[int] = list(range(num_pages - 1, -1, -1))
        self._pages: List[List[int]] = [[] for _ in range(batch_size)]
        self._tokens = [0] * batch_size  # that there is room for
        self._held = [0] * batch_size    # that have been appended, as far as the host has seen to it
        self._idle = [False] * batch_size
        self._captured = False           # a graph may append too

    @property
    def batch_size(self) -> int:
        return len(self._pages)

    def __repr__(self) -> str:
        pages, heads, size, _ = self.k_pages.shape
        return (f"PagedKVCache(pages={pages}, free={len(self._free)}, page_size={size}, kv_heads={heads}, "
                f"bits={self.bits}, batch_size={self.batch_size})")

    # -- pages ----------------------------------------------------------------------------------
    def reserve(self, tokens: Union[int, Sequence[int]]) -> None:
        """Make sure that every sequence (or each by its own number) has pages for so many tokens more than it
        holds. Raises, with nothing changed, if the pool or the table's rows have too few. One number for all leaves
        idle places out; one of its own, above 0, ends a place's being idle."""
        self._refuse_capture("reserve")
        if self._captured:
            self.sync()
        more = [0 if i else tokens for i in self._idle] if isinstance(tokens, int) else list(tokens)
        if len(more) != self.batch_size or min(more) < 0:
            raise ValueError(f"expected {self.batch_size} numbers of tokens, none negative")
        want = [max(t, h + n) for t, h, n in zip(self._tokens, self._held, more)]
        need = [-(-n // self.page_size) for n in want]
        missing = sum(max(0, n - len(p)) for n, p in zip(need, self._pages))
        if max(need) > self.max_pages or missing > len(self._free):
            raise RuntimeError(f"{missing} pages more are needed and {max(need)} for one sequence: the cache has "
                               f"{len(self._free)} free ones and room for {self.max_pages}")
        self._tokens = want
        self._idle = [i and n == 0 for i, n in zip(self._idle, more)]
        if missing:
            for p, n in zip(self._pages, need):
                while len(p) < n:
                    p.append(self._free.pop())
            self._write_table()

    def sync(self) -> None:
        """Read from the device how many tokens the sequences hold (after replays of captured steps, or a change of
        `lengths` from outside). Raises for one that is longer than its pages: tokens of it have been lost."""
        self._refuse_capture("sync")
        held = self.lengths.tolist()
        over = [b for b, (h, p) in enumerate(zip(held, self._pages)) if h > len(p) * self.page_size]
        if over:
            raise RuntimeError(f"sequences {over} have more tokens than their pages hold: replays went on behind what was "
                               "reserved, and those tokens are lost; set `lengths` back, or release the sequences")
        self._held = held
        self._tokens = [max(t, h) for t, h in zip(self._tokens, self._held)]

    def release(self, sequence: int, *, idle: bool = False) -> None:
        """Forget a sequence: its pages are free, and its place in the batch is empty. The next `append` (or `reserve`)
        begins another sequence there; with `idle`, `append` passes the place over until `reserve` is given a number
        of its own for it. Replays of captured steps pass over every place that has no pages."""
        self._refuse_capture("release")
        self._free.extend(reversed(self._pages[sequence]))
        self._pages[sequence] = []
        self._tokens[sequence] = self._held[sequence] = 0
        self._idle[sequence] = idle
        self.lengths[sequence] = 0
        self._write_table()

    def _write_table(self) -> None:
        rows = [[int(bool(p)), *p] + [-1] * (self.max_pages - len(p)) for p in self._pages]
        self._table.copy_(torch.tensor(rows, dtype=torch.int32))

    def _capturing(self) -> bool:
        return self.lengths.is_cuda and torch.cuda.is_current_stream_capturing()

    def _refuse_capture(self, what: str) -> None:
        """Before anything has changed: what the host does of it would be done, what the device does would not."""
        if self._capturing():
            raise RuntimeError(f"PagedKVCache.{what}() is not for a graph's capture: call it before")

    # -- kernels ----------------------------------------------------------------------------------
    def _scales(self) -> dict:
        return {} if self.bits == 16 else {"k_scales": self.k_scales, "v_scales": self.v_scales}

    def append(self, k: torch.Tensor, v: torch.Tensor, cos: Optional[torch.Tensor] = None,
               sin: Optional[torch.Tensor] = None, q: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """`ops.append_paged` of k / v (batch, S, heads, head_dim) behind what the sequences hold; pages are
        reserved for them if they have not been (not while a graph is captured). Rows of idle places are passed over.
        Returns the rotated queries."""
        if k.dim() != 4 or k.shape[0] != self.batch_size:
            raise ValueError(f"expected k ({self.batch_size}, tokens, heads, head_dim), got {tuple(k.shape)}")
        if k.dtype != self.dtype:
            raise TypeError(f"the cache is for {self.dtype}, got {k.dtype}")
        new, capturing = k.shape[1], self._capturing()
        if self._captured and not capturing:
            self.sync()
        held = [h if i else h + new for h, i in zip(self._held, self._idle)]
        if any(h > t for h, t in zip(held, self._tokens)):
            if capturing:
                raise RuntimeError("a captured step finds no room: reserve its replays' tokens before the capture")
            self.reserve(new)
        self.lengths.add_(self._in_use, alpha=new)
        try:
            out = ops.append_paged(k, v, self.k_pages, self.v_pages, self.block_table, self.lengths, cos=cos,
                                   sin=sin, q=q, **self._scales())
        except Exception:
            self.lengths.sub_(self._in_use, alpha=new)
            raise
        if capturing:
            self._captured = True  # nothing has run
        else:
            self._held = held
        return out

    def attend(self, q: torch.Tensor, *, scale: Optional[float] = None, window: Optional[Tuple[int, int]] = None,
               alibi_slopes: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of the last tokens q (batch, S, heads, head_dim) over the cache: `ops.attention_paged`
        for few of them, else the cache's rows packed (`ops.gather_paged`) and `ops.attention_packed`. Captured in a
        graph, the latter packs all that the batch may ever hold, since its replays may find more pages in use."""
        B, S, Hq, D = q.shape
        if S <= self.LONG:
            return ops.attention_paged(q, self.k_pages, self.v_pages, self.block_table, self.lengths, scale=scale,
                                       window=window, alibi_slopes=alibi_slopes, **self._scales())
        starts = self._starts()
        # room for all that the sequences' pages hold, whatever the host has seen of the lengths
        pages = sum(len(p) for p in self._pages)
        if self._capturing():
            pages = min(self.k_pages.shape[0], self.batch_size * self.max_pages)
        k, v = self._gather(starts, pages * self.page_size)
        rows = torch.arange(0, B * S + 1, S, dtype=torch.int32, device=q.device)
        out = ops.attention_packed(q.reshape(B * S, Hq, D), k, v, rows, starts, causal=True, scale=scale,
                                   window=None if window is None else (window[0], 0), alibi_slopes=alibi_slopes)
        return out.view(B, S, Hq, D)

    # Tokens to a sequence from which on the cache is read back for the kernel of packed sequences. attention_paged reads
    # the keys once for every 16 rows, tokens x query heads to a kv head; reading back costs the pages of all sequences,
    # in a captured step those of the pool. attention_paged / read back, us, 8 kv heads x 128 in 16 bits, 8 sequences of
    # 16000 keys: 1 query head to each, 16 tokens 97 / 361, 32 179 / 363, 64 339 / 366, 128 631 / 369; 4 heads, 8 tokens
    # 179 / 362, 16 338 / 369, 32 632 / 374; 64 sequences of 1000, 4 heads, 8 tokens 104 / 159, 16 184 / 161, 32 339 / 177;
    # one of 2000, 4 heads, 32 tokens 18 / 40, 64 32 / 43, 128 51 / 43.
    LONG = 32

    def gather(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """The sequences' keys and values one after the other, (tokens in all, heads, head_dim). Waits for the
        lengths."""
        return self._gather(self._starts(), int(self.lengths.sum()))

    def _starts(self) -> torch.Tensor:
        return torch.nn.functional.pad(self.lengths.cumsum(0, dtype=torch.int32), (1, 0))

    def _gather(self, starts: torch.Tensor, rows: int) -> Tuple[torch.Tensor, torch.Tensor]:
        return ops.gather_paged(self.k_pages, self.v_pages, self.block_table, starts, rows=rows, dtype=self.dtype,
                                **self._scales())
