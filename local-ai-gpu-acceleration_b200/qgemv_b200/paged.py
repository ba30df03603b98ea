"""Paged key-value cache for batched decode: torch front end of the qg_kv_pages entry points
(include/qgemv_b200.h has the formulas).

* `PagedCache` -- the key and value pools, seen as [page, head, place, dim], and the page
  list of every sequence.
* `qk_norm_rope_append` -- normalise and rotate new queries and keys, write keys and values
  to their slots.
* `AttentionPlan`, `attend` -- one new token per sequence attends to its sequence's slots.
* `evict` -- sequences are cut back to a budget of slots by the weight that `attend` summed.

Device memory and streams only; every computation happens in the library.  Inference only: no
call records a gradient, whatever its tensors require.  Every call takes
`stream` (default: the current one) and allocates what it returns on that stream, unless the
caller passes the output; tensors of other streams are the caller's to order.  Tensors that do
not fit raise ValueError (they are checked in csrc/qg_paged_torch.cpp: on small batches a call
takes as long as its checks), what the library refuses raises CudaError.
"""

from __future__ import annotations

import ctypes
from importlib.machinery import ExtensionFileLoader
from importlib.util import module_from_spec, spec_from_loader

import torch

from . import build as _build
from ._lib import CudaError, check, lib

QG_ERR_POSITION = 0x2
QG_ERR_PAGE = 0x4

PAIRS = {"adjacent": 0, "halves": 1}  # QG_PAIRS_*

_CALLS = None


def _calls():
    """The compiled front end, given the addresses of the library's entry points."""
    global _CALLS
    if _CALLS is None:
        path = str(_build.build_torch())
        loader = ExtensionFileLoader("qgemv_paged_torch", path)
        module = module_from_spec(spec_from_loader("qgemv_paged_torch", loader, origin=path))
        loader.exec_module(module)
        handle = lib()
        module.bind(*(ctypes.cast(fn, ctypes.c_void_p).value for fn in (
            handle.qg_qk_norm_rope_append, handle.qg_paged_attn, handle.qg_kv_evict)))
        module.bind8(*(ctypes.cast(fn, ctypes.c_void_p).value for fn in (
            handle.qg_qk_norm_rope_append8, handle.qg_kv_read8, handle.qg_paged_attn8)))
        _CALLS = module
    return _CALLS


class _MadeOnce:
    """What the library was told when an object was made holds for its calls: an attribute of the
    constructor's can be read, not replaced."""

    _replaceable: tuple[str, ...] = ()

    def __setattr__(self, name, value):
        if name in self.__dict__ and name not in self._replaceable:
            raise AttributeError(f"{type(self).__name__}.{name} cannot be replaced: calls use what the object was made of")
        object.__setattr__(self, name, value)


class PagedCache(_MadeOnce):
    """Pools `k` and `v` [pages, kv heads, page size, head dim] (fp16 or bf16, any strides
    with contiguous dims, the same for both) and `table` [sequences, pages per sequence]
    (int32).  The caller shares them: it hands out pages by writing into the table, and replaces
    or resizes none of the three.  Their memory stays while the cache, or a plan for it, does."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor):
        self.calls = _calls()
        self.held, self.pages_at = self.calls.cache(k, v, table)  # pages_at: its qg_kv_pages
        self.k, self.v, self.table = k, v, table
        self.device, self.dtype = k.device, k.dtype
        self.num_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.batch, self.table_pages = table.shape
        self.capacity = self.table_pages * self.page_size

    @staticmethod
    def empty(num_pages: int, n_kv_heads: int, page_size: int, head_dim: int, batch: int,
              table_pages: int, dtype=torch.float16, device="cuda") -> "PagedCache":
        """A cache of zeroed pools whose table names no page yet (every entry -1)."""
        shape = (num_pages, n_kv_heads, page_size, head_dim)
        return PagedCache(torch.zeros(shape, dtype=dtype, device=device),
                          torch.zeros(shape, dtype=dtype, device=device),
                          torch.full((batch, table_pages), -1, dtype=torch.int32, device=device))


def rope_table(rows: int, rot_dim: int, base: float = 500000.0, device="cuda") -> torch.Tensor:
    """[rows, rot_dim] fp32: the cosines, then the sines, of row * base^(-2i / rot_dim),
    angles in 64 bits."""
    inv = base ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


def qk_norm_rope_append(cache: PagedCache, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                        rope: torch.Tensor | None, positions: torch.Tensor, *,
                        slots: torch.Tensor | None = None, seqs: torch.Tensor | None = None,
                        q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None,
                        eps: float = 1e-5, pairs: str = "adjacent",
                        q_out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """qg_qk_norm_rope_append: q [tokens, q heads, dim], k and v [tokens, kv heads, dim] of one
    type (views of a fused projection are fine); returns the rotated queries."""
    if pairs not in PAIRS:
        raise ValueError("pairs: 'adjacent' or 'halves' is needed")
    code, q_out = cache.calls.append(cache.held, q, k, v, rope, positions, slots, seqs, q_norm, k_norm, eps,
                                     PAIRS[pairs], q_out, None if stream is None else stream.cuda_stream)
    if code != 0:
        raise CudaError("qg_qk_norm_rope_append", code)
    return q_out


class AttentionPlan(_MadeOnce):
    """The workspace of `attend` for a cache, a number of query heads and lengths up to
    max_len (default: all that a table row names).  Calls that may overlap need a plan each.
    `scale` is the scale of calls that name none."""

    _replaceable = ("scale",)

    def __init__(self, cache: PagedCache, n_q_heads: int, max_len: int | None = None,
                 weights: bool = False):
        self.cache, self.calls, self.n_q_heads, self.weights = cache, cache.calls, n_q_heads, weights
        self.max_len = cache.capacity if max_len is None else max_len
        n = ctypes.c_size_t(0)
        check("qg_paged_attn_workspace_bytes", cache.pages_at, n_q_heads, self.max_len, int(weights),
              ctypes.byref(n))
        self.workspace = torch.zeros(n.value, dtype=torch.uint8, device=cache.device)
        self.held = self.calls.plan(cache.held, n_q_heads, self.max_len, bool(weights), self.workspace)
        self.scale = cache.head_dim ** -0.5


def attend(plan: AttentionPlan, q: torch.Tensor, lens: torch.Tensor, *, window: int = 0,
           scale: float | None = None, out: torch.Tensor | None = None,
           lse: torch.Tensor | None = None, return_lse: bool = False,
           weight_in: torch.Tensor | None = None, weight_out: torch.Tensor | None = None,
           stream=None):
    """qg_paged_attn: q [sequences, q heads, dim] attends to lens[b] slots of sequence b (scale
    defaults to dim^-1/2); returns out like q, or (out, lse [sequences, q heads]).
    weight_out [sequences, kv heads, >= max_len] receives weight_in plus each slot's shares
    (a plan with weights; weight_in may be weight_out)."""
    code, out, lse = plan.calls.attend(plan.held, q, lens, window, plan.scale if scale is None else scale, out,
                                       lse, bool(return_lse), weight_in, weight_out,
                                       None if stream is None else stream.cuda_stream)
    if code != 0:
        raise CudaError("qg_paged_attn", code)
    return out if lse is None else (out, lse)


def evict(cache: PagedCache, lens: torch.Tensor, weight: torch.Tensor, budget: int, *, sink: int = 0,
          recent: int = 0, new_table: torch.Tensor | None = None, lens_out: torch.Tensor | None = None,
          weight_out: torch.Tensor | None = None, kept: torch.Tensor | None = None, stream=None):
    """qg_kv_evict: keep `budget` slots per kv head of every longer sequence -- the first `sink`,
    the last `recent`, and the heaviest between them by weight [sequences, kv heads, >= longest
    length].  Rows move to the front of the same pages, lens and weight are updated; or, with
    new_table [sequences, pages], to those pages, the new weights to weight_out (needed then; it
    may be weight) and lens left as it is.  The work is sized for the rows of weight, so rows not
    much wider than the longest length are the fastest; into other pages takes less time than in
    place.  Returns (kept [sequences, kv heads, budget], new lens)."""
    code, kept, lens_out = cache.calls.evict(cache.held, lens, weight, budget, sink, recent, new_table, lens_out,
                                             weight_out, kept, None if stream is None else stream.cuda_stream)
    if code != 0:
        raise CudaError("qg_kv_evict", code)
    return kept, lens_out
