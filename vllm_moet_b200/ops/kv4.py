"""4-bit paged K/V cache for layers with K/V heads of their own (grouped-query attention).

The engine's NVFP4 cache row (``formats/kv_nvfp4.py``) is the MLA latent; this cache holds
full K and V rows of grouped-query layers that a user brings (the engine's own layers are MLA), in
4.5 bits a value: e2m1 codes with one e4m3 scale per 16 values (``formats/kv4.py`` has the
byte layout and the golden encoder).  It can be read whole or by chosen pages:

    cache = KV4Cache(num_pages, num_kv_heads, head_dim)
    cache.append(k, v, slots)                                    # quantise rows into their slots
    k, v = cache.read(slots)                                     # rows back, in 16 bits
    pages = cache.select(q, cu_q, seq_lens, block_table, 64)     # 64 pages per token and K/V head
    out = cache.attend(q, cu_q, seq_lens, block_table, scale)    # over every page
    out = cache.attend(q, cu_q, seq_lens, block_table, scale, pages=pages)

A batch is described as elsewhere in the engine: rows of all sequences in one tensor, row
offsets ``cu_q`` int32 [B + 1], ``seq_lens`` int32 [B] positions held per sequence including
the rows' own (append first), ``block_table`` int32 [B, W] page per 64 positions.  Row i of a
sequence's n sits at position ``seq_len - n + i`` and sees the positions up to its own.

All calls run on the current CUDA stream, never synchronise and can be captured in a CUDA
graph.  Errors that only the device can see (a slot, page, length or row
offset out of range, a value that is not finite) set ``cache.status``, as the engine's other kernels do; ``cache.check()`` raises.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import native

PAGE = 64
HEAD_DIMS = (64, 128, 256)
_STATUS = {1: "a slot, page, length or row offset out of range", 2: "a wait on the device ran out", 3: "a sequence with more rows than max_q",
           4: "a key or value that is not finite (NaN is held as 0, infinities as the largest value)"}


class KV4Cache:
    """Pages of 64 positions of ``num_kv_heads`` heads, held in 4 bits.

    ``k_exp`` / ``v_exp``: an element is e2m1 * e4m3 scale * 2^exp; the default reaches 42 in
    steps fine enough for normalised keys and values.  Larger values saturate."""

    _tries = 1 << 22        # of a wait on the device (about a second) before the kernel gives up and sets the status

    def __init__(self, num_pages: int, num_kv_heads: int, head_dim: int, device="cuda", k_exp: int = -6,
                 v_exp: int = -6):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if num_pages < 1 or num_kv_heads < 1:
            raise ValueError("num_pages and num_kv_heads must be at least 1")
        if num_kv_heads > 65535:
            raise ValueError("num_kv_heads must be at most 65535 (a grid's second dimension)")
        if not (-14 <= k_exp <= 4 and -14 <= v_exp <= 4):
            raise ValueError("k_exp and v_exp must lie in [-14, 4] (what f16 holds exactly)")
        device = torch.device(device)
        if device.type != "cuda":
            raise ValueError(f"KV4Cache runs on a CUDA device, got {device}")
        self._C = native()
        self.num_pages, self.num_kv_heads, self.head_dim = num_pages, num_kv_heads, head_dim
        self.k_exp, self.v_exp = k_exp, v_exp
        self.pages = torch.zeros(num_pages, num_kv_heads, 72 * head_dim, dtype=torch.uint8, device=device)
        # page bounds: ceil(max / unit), floor(min / unit) of each key channel over the page's rows
        self.bounds = torch.zeros(num_pages, num_kv_heads, 2, head_dim, dtype=torch.int8, device=device)
        self.unit = torch.ones(num_pages, num_kv_heads, dtype=torch.float32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.device = self.pages.device

    @property
    def bytes_per_token(self) -> int:
        return self.num_kv_heads * 72 * self.head_dim // PAGE

    def check(self) -> None:
        """Raise if a kernel has reported an error (synchronises).  The first error stays until ``status`` is zeroed."""
        s = int(self.status)
        if s:
            raise RuntimeError(f"kv4: {_STATUS.get(s, f'status {s}')}")

    # ------------------------------------------------------------------ operators
    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantise rows k, v [T, num_kv_heads, head_dim] (bf16 or f16, inner stride 1) into slots
        ``page * 64 + offset``; a negative slot skips its row.  Finite values past 2688 * 2^exp (42 by default) are
        held as the largest value without a report; NaN and infinities set the status.  The bounds of every page touched
        are recomputed.  Rows may come in any order, but no slot twice in one call."""
        self._C.kv4_append(k, v, slots, self.pages, self.bounds, self.unit, self.status, self.k_exp, self.v_exp)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
        """The rows of ``slots`` as 16-bit values (exact: six significant bits); zeros where a slot is negative."""
        return self._C.kv4_read(slots, dtype, self.pages, self.bounds, self.unit, self.status, self.k_exp, self.v_exp)

    def select(self, q: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor,
               budget: int, *, first: int = 1, last: int = 2, max_q: Optional[int] = None) -> torch.Tensor:
        """The ``budget`` pages that each row and K/V head should attend to -> int32 [rows, K/V heads, budget],
        logical page indices in ascending order, -1 after the last where a row has fewer pages.

        The first ``first`` and the last ``last`` (>= 1) pages up to the row's own are always taken; the
        others compete by an estimate of their largest logit for a positive scale: the upper bound that
        the page's bounds give for the query rounded to 8 bits.  It is computed exactly, so equal inputs give
        equal choices on every rank, and ties go to the lowest page.  Where the table is wider than ``budget``,
        rows * K/V heads * W floats of workspace are taken: give a table as wide as the longest sequence.
        A row past ``max_q`` of its sequence may get no page, which sets the status.  Needs the rows' own
        positions appended: pages before a row's last one must be complete."""
        return self._C.kv4_select(q, cu_q, seq_lens, block_table, budget, first, last, -1 if max_q is None else max_q,
                                  self.pages, self.bounds, self.unit, self.status)

    def attend(self, q: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor,
               scale: float, *, max_q: Optional[int] = None, window: int = 0, pages: Optional[torch.Tensor] = None,
               return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
        """softmax(scale * q k^T) v for every row of the batch -> [rows, heads, head_dim] in q's type.

        ``max_q``: the most rows of one sequence (default: all rows); it sizes the work and chooses between
        two kernels for the whole batch, so give it where it is known, and serve long prompt chunks and decode
        rows in calls of their own.  Rows past it may come out as zeros, which sets the status.  ``window`` > 0:
        only the last ``window`` positions up to the row's own.  ``pages`` int32 [rows, K/V heads, n]: only the
        positions of these pages of the row's sequence (logical indices, each at most once, -1 for
        none), as :meth:`select` gives them.  A row that sees nothing is zeros.  ``return_lse``:
        also the natural log-sum-exp [rows, heads] f32 (-inf for a row that sees nothing)."""
        out, lse = self._C.kv4_attend(q, cu_q, seq_lens, block_table, scale, -1 if max_q is None else max_q, window, pages,
                                      return_lse, self.pages, self.bounds, self.unit, self.status, self.k_exp, self.v_exp,
                                      self._tries)
        return (out, lse) if return_lse else out
