"""Paged key-value cache in 8 bits: torch front end of the qg_kv_pages8 entry points
(include/qgemv_b200.h has the formulas).

* `PagedCache8` -- pools of e4m3 codes, seen as [page, head, place, dim], the scales of their
  blocks, [page, head, block of the page], and the page list of every sequence.
* `qk_norm_rope_append` -- normalise and rotate new queries and keys, quantise keys and values
  into the blocks of their slots.
* `read` -- rows of the cache as the 16- or 32-bit values that they stand for.
* `AttentionPlan8`, `attend` -- the new tokens of every sequence, one or many, attend to its
  slots: all of them, or a window and the first few.

A call has its rows sequence after sequence: `offsets` [sequences + 1] (int32, on the device) says
where each begins, None stands for one row a sequence.  `lens` [sequences] counts a sequence's slots
with its new tokens, which are the last of them.  Rows outside offsets[0] to offsets[-1] belong to no
sequence and are left alone; in a tensor that the call makes they hold anything.

Streams, outputs, lifetimes and errors are those of `paged`; inference only.
"""

from __future__ import annotations

import ctypes

import torch

from ._lib import CudaError, check
from .paged import PAIRS, _calls, _MadeOnce, rope_table  # noqa: F401


class PagedCache8(_MadeOnce):
    """Pools `k` and `v` [pages, kv heads, page size, head dim] (float8_e4m3fn, any strides of whole
    16 bytes with contiguous dims, the same for both), `k_scale` and `v_scale` [pages, kv heads,
    blocks of a page] (float32) and `table` [sequences, pages per sequence] (int32).  A block is 16,
    32, 64 or 128 slots and divides a page.  The caller hands out pages by writing into the table."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                 table: torch.Tensor):
        self.calls = _calls()
        self.held, self.pages_at, self.block = self.calls.cache8(k, v, k_scale, v_scale, table)
        self.k, self.v, self.k_scale, self.v_scale, self.table = k, v, k_scale, v_scale, table
        self.device = k.device
        self.num_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.batch, self.table_pages = table.shape
        self.capacity = self.table_pages * self.page_size

    @staticmethod
    def empty(num_pages: int, n_kv_heads: int, page_size: int, head_dim: int, batch: int,
              table_pages: int, block: int = 32, device="cuda") -> "PagedCache8":
        """A cache of zeroed pools whose table names no page yet (every entry -1)."""
        if block < 1 or page_size % block != 0:
            raise ValueError("block: a part of a page is needed")
        shape, blocks = (num_pages, n_kv_heads, page_size, head_dim), (num_pages, n_kv_heads, page_size // block)
        return PagedCache8(*(torch.zeros(shape, dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
                             for _ in range(2)),
                           *(torch.zeros(blocks, device=device) for _ in range(2)),
                           torch.full((batch, table_pages), -1, dtype=torch.int32, device=device))


def qk_norm_rope_append(cache: PagedCache8, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        rope: torch.Tensor | None, positions: torch.Tensor, lens: torch.Tensor, *,
                        offsets: torch.Tensor | None = None, q_norm: torch.Tensor | None = None,
                        k_norm: torch.Tensor | None = None, eps: float = 1e-5, pairs: str = "adjacent",
                        q_out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """qg_qk_norm_rope_append8: q [tokens, q heads, dim], k and v [tokens, kv heads, dim] of one
    type (views of a fused projection are fine), `lens` the lengths with these tokens; returns
    the rotated queries."""
    if pairs not in PAIRS:
        raise ValueError("pairs: 'adjacent' or 'halves' is needed")
    code, q_out = cache.calls.append8(cache.held, q, k, v, rope, positions, lens, offsets, q_norm, k_norm, eps,
                                      PAIRS[pairs], q_out, None if stream is None else stream.cuda_stream)
    if code != 0:
        raise CudaError("qg_qk_norm_rope_append8", code)
    return q_out


def read(cache: PagedCache8, starts: torch.Tensor, offsets: torch.Tensor, tokens: int, *,
         dtype: torch.dtype = torch.float16, k_out: torch.Tensor | None = None,
         v_out: torch.Tensor | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """qg_kv_read8: keys and values [tokens, kv heads, dim] of `dtype`; rows offsets[b] on are the
    slots from starts[b] [sequences] on of sequence b."""
    code, k_out, v_out = cache.calls.read8(cache.held, starts, offsets, tokens, dtype, k_out, v_out,
                                           None if stream is None else stream.cuda_stream)
    if code != 0:
        raise CudaError("qg_kv_read8", code)
    return k_out, v_out


class AttentionPlan8(_MadeOnce):
    """The workspace of `attend` for a cache, a number of query heads and calls of up to max_tokens
    rows (default: one a sequence).  Calls that may overlap need a plan each.  `scale` is the
    scale of calls that name none."""

    _replaceable = ("scale",)

    def __init__(self, cache: PagedCache8, n_q_heads: int, max_tokens: int | None = None):
        self.cache, self.calls, self.n_q_heads = cache, cache.calls, n_q_heads
        self.max_tokens = cache.batch if max_tokens is None else max_tokens
        n = ctypes.c_size_t(0)
        check("qg_paged_attn8_workspace_bytes", cache.pages_at, n_q_heads, self.max_tokens, ctypes.byref(n))
        self.workspace = torch.zeros(n.value, dtype=torch.uint8, device=cache.device)
        self.held = self.calls.plan8(cache.held, n_q_heads, self.max_tokens, self.workspace)
        self.scale = cache.head_dim ** -0.5


def attend(plan: AttentionPlan8, q: torch.Tensor, lens: torch.Tensor, *, offsets: torch.Tensor | None = None,
           window: int = 0, sink: int = 0, scale: float | None = None, out: torch.Tensor | None = None,
           lse: torch.Tensor | None = None, return_lse: bool = False, stream=None):
    """qg_paged_attn8: q [tokens, q heads, dim]; each new token attends to the slots up to its own
    (with `window`, the last `window` of them and the first `sink`); scale defaults to dim^-1/2.
    Returns out like q, or (out, lse [tokens, q heads])."""
    code, out, lse = plan.calls.attend8(plan.held, q, lens, offsets, window, sink,
                                        plan.scale if scale is None else scale, out, lse, bool(return_lse),
                                        None if stream is None else stream.cuda_stream)
    if code != 0:
        raise CudaError("qg_paged_attn8", code)
    return out if lse is None else (out, lse)
