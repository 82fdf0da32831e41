"""4-bit paged K/V cache for layers with K/V heads of their own (grouped-query attention).

The engine's NVFP4 cache row (``formats/kv_nvfp4.py``) is the MLA latent; this cache holds
full K and V rows of grouped-query layers, such as drafters trained beside an MLA target, in
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
graph.  Errors that only the device can see (a slot or page out of range, a value that is not
finite) set ``cache.status``, as the engine's other kernels do; ``cache.check()`` raises.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import native

PAGE = 64
HEAD_DIMS = (64, 128, 256)
# query rows of one sequence and K/V head above which attention runs on the tcgen05 kernel
PROMPT_ROWS = 64
_STATUS = {1: "a slot or page out of range", 2: "a wait on the device ran out", 3: "bad size",
           4: "a key or value that is not finite (NaN is held as 0, infinities as the largest value)"}

# parts of split tiles (kv4_attend), by stream: calls on one stream run one after the other
_workspaces: dict = {}


def _workspace(device: torch.device, floats: int, ints: int) -> Tuple[torch.Tensor, torch.Tensor]:
    key = (device.index, torch.cuda.current_stream(device).cuda_stream)
    part, split = _workspaces.get(key, (None, None))
    if part is None or part.numel() < floats:
        part = torch.empty(floats, dtype=torch.float32, device=device)
        split = torch.empty(ints, dtype=torch.int32, device=device)
        if not torch.cuda.is_current_stream_capturing():      # a captured graph owns its workspace
            _workspaces[key] = (part, split)
    return part, split


class KV4Cache:
    """Pages of 64 positions of ``num_kv_heads`` heads, held in 4 bits.

    ``k_exp`` / ``v_exp``: an element is e2m1 * e4m3 scale * 2^exp; the default reaches 42 in
    steps fine enough for normalised keys and values.  Larger values saturate."""

    def __init__(self, num_pages: int, num_kv_heads: int, head_dim: int, device="cuda", k_exp: int = -6,
                 v_exp: int = -6):
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"head_dim must be one of {HEAD_DIMS}, got {head_dim}")
        if num_pages < 1 or num_kv_heads < 1:
            raise ValueError("num_pages and num_kv_heads must be at least 1")
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
        """Raise if a kernel has reported an error (synchronises)."""
        s = int(self.status)
        if s:
            raise RuntimeError(f"kv4: {_STATUS.get(s, f'status {s}')}")

    # ------------------------------------------------------------------ checks
    def _need(self, ok: bool, what: str) -> None:
        if not ok:
            raise ValueError(f"kv4: {what}")

    def _slots(self, slots: torch.Tensor, T: Optional[int] = None) -> None:
        self._need(slots.device == self.device and slots.dtype == torch.int64 and slots.dim() == 1
                   and slots.is_contiguous() and (T is None or slots.shape[0] == T),
                   "slots must be a contiguous int64 tensor with one slot per row, on the cache's device")

    def _batch(self, q, cu_q, seq_lens, block_table, max_q) -> int:
        H, D = self.num_kv_heads, self.head_dim
        self._need(q.device == self.device and q.dtype in (torch.bfloat16, torch.float16) and q.dim() == 3
                   and q.shape[2] == D and q.stride(2) == 1, f"q must be bf16 or f16 [rows, heads, {D}], inner stride 1")
        self._need(q.shape[1] >= H and q.shape[1] % H == 0, f"q's heads must be a multiple of the {H} K/V heads")
        for name, x, n in (("cu_q", cu_q, seq_lens.shape[0] + 1), ("seq_lens", seq_lens, seq_lens.shape[0])):
            self._need(x.device == self.device and x.dtype == torch.int32 and x.dim() == 1 and x.is_contiguous()
                       and x.shape[0] == n, f"{name} must be a contiguous int32 tensor [{n}]")
        self._need(block_table.device == self.device and block_table.dtype == torch.int32 and block_table.dim() == 2
                   and block_table.is_contiguous() and block_table.shape[0] == seq_lens.shape[0]
                   and block_table.shape[1] >= 1, "block_table must be a contiguous int32 tensor [sequences, pages >= 1]")
        if max_q is None:
            max_q = q.shape[0]
        self._need(max_q >= 1 or q.shape[0] == 0, "max_q must be at least 1")
        return max_q

    # ------------------------------------------------------------------ operators
    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantise rows k, v [T, num_kv_heads, head_dim] (bf16 or f16, inner stride 1) into slots
        ``page * 64 + offset``; a negative slot skips its row.  The bounds of every page touched
        are recomputed.  Rows may come in any order, but no slot twice in one call."""
        T, H, D = slots.shape[0], self.num_kv_heads, self.head_dim
        self._slots(slots)
        for x in (k, v):
            self._need(x.device == self.device and x.shape == (T, H, D) and x.dtype == k.dtype
                       and x.dtype in (torch.bfloat16, torch.float16) and x.stride(2) == 1,
                       f"k and v must be bf16 or f16 [{T}, {H}, {D}] of one type, inner stride 1, on the cache's device")
        self._C.kv4_append(k, v, slots, self.pages, self.bounds, self.unit, self.k_exp, self.v_exp, self.status)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
        """The rows of ``slots`` as 16-bit values (exact: six significant bits); zeros where a slot is negative."""
        self._slots(slots)
        self._need(dtype in (torch.bfloat16, torch.float16), "read gives bf16 or f16")
        shape = (slots.shape[0], self.num_kv_heads, self.head_dim)
        k, v = (torch.empty(shape, dtype=dtype, device=self.device) for _ in range(2))
        self._C.kv4_read(slots, self.pages, self.k_exp, self.v_exp, k, v, self.status)
        return k, v

    def select(self, q: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor,
               budget: int, *, first: int = 1, last: int = 2, max_q: Optional[int] = None) -> torch.Tensor:
        """The ``budget`` pages that each row and K/V head should attend to -> int32 [rows, K/V heads, budget],
        logical page indices in ascending order, -1 after the last where a row has fewer pages.

        The first ``first`` and the last ``last`` (>= 1) pages up to the row's own are always taken; the
        others compete by an upper bound on their logits that is computed exactly, so equal inputs give
        equal choices on every rank, and ties go to the lowest page.  Needs the rows' own positions
        appended: pages before a row's last one must be complete."""
        max_q = self._batch(q, cu_q, seq_lens, block_table, max_q)
        self._need(first >= 0 and last >= 1 and first + last <= budget,
                   f"need first >= 0, last >= 1 and first + last <= budget, got {first}, {last}, {budget}")
        T, H, W = q.shape[0], self.num_kv_heads, block_table.shape[1]
        pages = torch.empty(T, H, budget, dtype=torch.int32, device=self.device)
        score = torch.empty(T * H * W if W > budget else 0, dtype=torch.float32, device=self.device)
        if T:
            self._C.kv4_select(q, cu_q, seq_lens, block_table, self.bounds, self.unit, max_q, first, last, score,
                               pages, self.status)
        return pages

    def attend(self, q: torch.Tensor, cu_q: torch.Tensor, seq_lens: torch.Tensor, block_table: torch.Tensor,
               scale: float, *, max_q: Optional[int] = None, window: int = 0, pages: Optional[torch.Tensor] = None,
               return_lse: bool = False) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
        """softmax(scale * q k^T) v for every row of the batch -> [rows, heads, head_dim] in q's type.

        ``max_q``: the most rows of one sequence (default: all rows).  ``window`` > 0: only the last
        ``window`` positions up to the row's own.  ``pages`` int32 [rows, K/V heads, n]: only the
        positions of these pages of the row's sequence (logical indices, each at most once, -1 for
        none), as :meth:`select` gives them.  A row that sees nothing is zeros.  ``return_lse``:
        also the natural log-sum-exp [rows, heads] f32 (-inf for a row that sees nothing)."""
        max_q = self._batch(q, cu_q, seq_lens, block_table, max_q)
        self._need(window >= 0, "window must be >= 0")
        T, Hq = q.shape[0], q.shape[1]
        if pages is not None:
            self._need(pages.device == self.device and pages.dtype == torch.int32 and pages.is_contiguous()
                       and pages.dim() == 3 and pages.shape[:2] == (T, self.num_kv_heads) and pages.shape[2] >= 1,
                       f"pages must be a contiguous int32 tensor [{T}, {self.num_kv_heads}, n >= 1]")
        if q.stride(0) % 8 or q.stride(1) % 8 or q.data_ptr() % 16:      # the kernel copies rows 16 bytes at a time
            q = q.clone(memory_format=torch.contiguous_format)
        out = torch.empty(T, Hq, self.head_dim, dtype=q.dtype, device=self.device)
        lse = torch.empty(T, Hq, dtype=torch.float32, device=self.device) if return_lse else None
        if T and pages is None and max_q * (Hq // self.num_kv_heads) > PROMPT_ROWS:
            self._C.kv4_prompt(q, cu_q, seq_lens, block_table, self.pages, scale, max_q, window, self.k_exp, self.v_exp,
                               out, lse, self.status)
        elif T:
            part, split = _workspace(self.device, *self._C.kv4_attend_workspace(
                Hq // self.num_kv_heads, self.head_dim, max_q, pages is not None))
            self._C.kv4_attend(q, cu_q, seq_lens, block_table, self.pages, pages, scale, max_q, window, self.k_exp,
                               self.v_exp, out, lse, part, split, self.status)
        return (out, lse) if return_lse else out
