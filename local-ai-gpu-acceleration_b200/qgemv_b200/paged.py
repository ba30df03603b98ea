"""Paged key-value cache for batched decode: torch front end of the qg_kv_pages entry points
(include/qgemv_b200.h has the formulas).

* `PagedCache` -- the key and value pools, seen as [page, head, place, dim], and the page
  list of every sequence.
* `qk_norm_rope_append` -- normalise and rotate new queries and keys, write keys and values
  to their slots.
* `AttentionPlan`, `attend` -- one new token per sequence attends to its sequence's slots.
* `evict` -- sequences are cut back to a budget of slots by the weight that `attend` summed.

Device memory and streams only; every computation happens in the library.  Every call takes
`stream` (default: the current one) and allocates what it returns on that stream, unless the
caller passes the output; tensors of other streams are the caller's to order.
"""

from __future__ import annotations

import ctypes
from ctypes import c_float, c_int, c_uint32, c_uint64, c_void_p

import torch

from ._lib import CudaError, lib

QG_ERR_POSITION = 0x2
QG_ERR_PAGE = 0x4

DTYPE_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # qg_dtype
PAIRS = {"adjacent": 0, "halves": 1}


class KvPagesC(ctypes.Structure):
    _fields_ = [("k", c_void_p), ("v", c_void_p), ("dtype", c_int),
                ("num_pages", c_uint32), ("page_size", c_uint32), ("n_kv_heads", c_uint32),
                ("head_dim", c_uint32), ("page_stride", c_uint64), ("head_stride", c_uint64),
                ("slot_stride", c_uint64), ("table", c_void_p), ("batch", c_uint32),
                ("table_pages", c_uint32), ("table_stride", c_uint32)]


class AppendC(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("k", c_void_p), ("v", c_void_p), ("q_out", c_void_p),
                ("dtype", c_int), ("tokens", c_uint32), ("n_q_heads", c_uint32),
                ("q_stride", c_uint64), ("k_stride", c_uint64), ("v_stride", c_uint64),
                ("q_out_stride", c_uint64), ("q_norm", c_void_p), ("k_norm", c_void_p),
                ("eps", c_float), ("rope", c_void_p), ("rope_rows", c_uint32),
                ("rot_dim", c_uint32), ("pairs", c_int), ("positions", c_void_p),
                ("slots", c_void_p), ("seqs", c_void_p)]


class AttnC(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("out", c_void_p), ("dtype", c_int), ("n_q_heads", c_uint32),
                ("q_stride", c_uint64), ("out_stride", c_uint64), ("lens", c_void_p),
                ("max_len", c_uint32), ("window", c_uint32), ("scale", c_float),
                ("lse", c_void_p), ("weight_in", c_void_p), ("weight_out", c_void_p),
                ("weight_stride", c_uint32)]


class EvictC(ctypes.Structure):
    _fields_ = [("lens", c_void_p), ("lens_out", c_void_p), ("weight", c_void_p),
                ("weight_out", c_void_p), ("max_len", c_uint32), ("weight_stride", c_uint32),
                ("budget", c_uint32), ("sink", c_uint32), ("recent", c_uint32),
                ("kept", c_void_p), ("new_table", c_void_p), ("new_table_pages", c_uint32),
                ("new_table_stride", c_uint32)]


def _fail(message: str):
    raise ValueError(message)


# The checks below run on every call and on small batches take as long as the kernels, so each
# reads an attribute once and calls nothing it does not need.
_F32, _I32 = torch.float32, torch.int32
_device_now = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream
_byref = ctypes.byref
_empty_like = torch.empty_like


def _call(fn, index: int, *args) -> None:
    """Call an entry point with device `index` current."""
    if _device_now() != index:
        with torch.cuda.device(index):
            code = fn(*args)
    else:
        code = fn(*args)
    if code != 0:
        raise CudaError(fn.__name__, code)


def _new_ints(shape: tuple, like: torch.Tensor, stream) -> torch.Tensor:
    """The same of another shape."""
    if stream is None:
        return like.new_empty(shape)
    with torch.cuda.stream(stream):
        return like.new_empty(shape)


def _like(t: torch.Tensor, stream) -> torch.Tensor:
    """A new tensor like t, on the stream that will write it."""
    if stream is None:
        return _empty_like(t)
    with torch.cuda.stream(stream):
        return _empty_like(t)


def _ints(t: torch.Tensor, n: int, name: str, index: int) -> int:
    """Address of a contiguous int32 tensor of n entries."""
    if t.dtype is not _I32 or t.numel() != n or t.get_device() != index or not t.is_contiguous():
        _fail(f"{name}: a contiguous int32 tensor of {n} entries on cuda:{index} is needed")
    return t.data_ptr()


def _floats(t: torch.Tensor, shape: tuple, name: str, index: int) -> int:
    """Address of a contiguous fp32 tensor of a shape."""
    if t.dtype is not _F32 or t.shape != shape or t.get_device() != index or not t.is_contiguous():
        _fail(f"{name}: a contiguous float32 tensor of shape {shape} on cuda:{index} is needed")
    return t.data_ptr()


def _heads(t: torch.Tensor, shape: tuple, dtype, name: str, index: int) -> int:
    """Stride from row to row of a [rows, heads, dim] tensor whose rows are contiguous."""
    if t.shape != shape or t.dtype is not dtype or t.get_device() != index:
        _fail(f"{name}: a {dtype} tensor of shape {shape} on cuda:{index} is needed")
    rows, heads, dim = shape
    row, head, one = t.stride()
    if one != 1 or (head != dim and heads > 1):
        _fail(f"{name}: the heads of one row must be contiguous")
    return row if rows > 1 else heads * dim


class PagedCache:
    """Pools `k` and `v` [pages, kv heads, page size, head dim] (fp16 or bf16, any strides
    with contiguous dims, the same for both) and `table` [sequences, pages per sequence]
    (int32).  The caller owns them: it hands out pages by writing the table."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor):
        def steps(t):  # a dimension of one entry has no step
            return [s if n > 1 else 0 for s, n in zip(t.stride(), t.shape)]

        if k.dim() != 4 or k.shape != v.shape or steps(k) != steps(v) or k.dtype != v.dtype:
            _fail("k and v: two [pages, heads, page size, dim] tensors of one type and layout are needed")
        if not k.is_cuda or k.device != v.device or k.device != table.device:
            _fail("k, v and table have to be on one CUDA device (there is no CPU path)")
        if k.dtype not in (torch.float16, torch.bfloat16) or steps(k)[3] != 1:
            _fail("k and v: float16 or bfloat16 with contiguous dims are needed")
        if table.dtype != torch.int32 or table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
            _fail("table: an int32 tensor [sequences, pages per sequence] is needed")
        self.k, self.v, self.table = k, v, table
        self.device, self.dtype, self.index = k.device, k.dtype, k.get_device()
        self.num_pages, self.n_kv_heads, self.page_size, self.head_dim = k.shape
        self.batch, self.table_pages = table.shape
        self.capacity = self.table_pages * self.page_size
        stride = steps(k)
        self.c = KvPagesC(k.data_ptr(), v.data_ptr(), DTYPE_CODES[k.dtype], self.num_pages,
                          self.page_size, self.n_kv_heads, self.head_dim, stride[0], stride[1],
                          stride[2], table.data_ptr(), self.batch, self.table_pages,
                          table.stride(0) if self.batch > 1 else self.table_pages)
        self._ref = ctypes.byref(self.c)

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
    index, dim, kv, dtype = cache.index, cache.head_dim, cache.n_kv_heads, q.dtype
    if dtype not in DTYPE_CODES or q.dim() != 3:
        _fail("q: a [tokens, heads, dim] tensor of float32, float16 or bfloat16 is needed")
    if pairs not in PAIRS:
        _fail("pairs is 'adjacent' or 'halves'")
    tokens, heads, _ = q.shape
    q_shape, kv_shape = (tokens, heads, dim), (tokens, kv, dim)
    q_stride = _heads(q, q_shape, dtype, "q", index)
    if q_out is None:
        q_out, out_stride = _like(q, stream), heads * dim
    else:
        out_stride = _heads(q_out, q_shape, dtype, "q_out", index)
    rows, rot = (0, 0) if rope is None else rope.shape
    a = AppendC(q.data_ptr(), k.data_ptr(), v.data_ptr(), q_out.data_ptr(), DTYPE_CODES[dtype],
                tokens, heads, q_stride, _heads(k, kv_shape, dtype, "k", index),
                _heads(v, kv_shape, dtype, "v", index), out_stride,
                None if q_norm is None else _floats(q_norm, (dim,), "q_norm", index),
                None if k_norm is None else _floats(k_norm, (dim,), "k_norm", index), eps,
                None if rope is None else _floats(rope, (rows, rot), "rope", index), rows, rot,
                PAIRS[pairs], _ints(positions, tokens, "positions", index),
                None if slots is None else _ints(slots, tokens, "slots", index),
                None if seqs is None else _ints(seqs, tokens, "seqs", index))
    _call(lib().qg_qk_norm_rope_append, index, cache._ref, _byref(a),
          _raw_stream(index) if stream is None else stream.cuda_stream)
    return q_out


class AttentionPlan:
    """The workspace of `attend` for a cache, a number of query heads and lengths up to
    max_len (default: all that a table row names).  Calls that may overlap need a plan each."""

    def __init__(self, cache: PagedCache, n_q_heads: int, max_len: int | None = None,
                 weights: bool = False):
        self.cache, self.n_q_heads, self.weights = cache, n_q_heads, weights
        self.shape = (cache.batch, n_q_heads, cache.head_dim)
        self.max_len = cache.capacity if max_len is None else max_len
        n = ctypes.c_size_t(0)
        _call(lib().qg_paged_attn_workspace_bytes, cache.index, cache._ref, n_q_heads, self.max_len,
              int(weights), _byref(n))
        self.workspace = torch.zeros(n.value, dtype=torch.uint8, device=cache.device)
        self.workspace_at = self.workspace.data_ptr()
        self.lse = torch.empty(cache.batch, n_q_heads, device=cache.device)  # what new ones are made like


def attend(plan: AttentionPlan, q: torch.Tensor, lens: torch.Tensor, *, window: int = 0,
           scale: float | None = None, out: torch.Tensor | None = None,
           lse: torch.Tensor | None = None, return_lse: bool = False,
           weight_in: torch.Tensor | None = None, weight_out: torch.Tensor | None = None,
           stream=None):
    """qg_paged_attn: q [sequences, q heads, dim] attends to lens[b] slots of sequence b (scale
    defaults to dim^-1/2); returns out like q, or (out, lse [sequences, q heads]).
    weight_out [sequences, kv heads, >= max_len] receives weight_in plus each slot's shares
    (a plan with weights; weight_in may be weight_out)."""
    cache, shape, dtype = plan.cache, plan.shape, q.dtype
    index = cache.index
    batch, heads, dim = shape
    if dtype not in DTYPE_CODES:
        _fail("q: float32, float16 or bfloat16 is needed")
    if window < 0:
        _fail("window is a number of slots, 0 for all")
    q_stride = _heads(q, shape, dtype, "q", index)
    if out is None:
        out, out_stride = _like(q, stream), heads * dim
    else:
        out_stride = _heads(out, shape, dtype, "out", index)
    if lse is not None:
        _floats(lse, (batch, heads), "lse", index)
    elif return_lse:
        lse = _like(plan.lse, stream)
    width, w_in, w_out = 0, None, None
    if weight_out is not None:
        if not plan.weights:
            _fail("weight_out needs a plan with weights")
        width = weight_out.shape[-1]
        w_out = _floats(weight_out, (batch, cache.n_kv_heads, width), "weight_out", index)
        if weight_in is not None:
            w_in = _floats(weight_in, (batch, cache.n_kv_heads, width), "weight_in", index)
    elif weight_in is not None:
        _fail("weight_in without weight_out")
    a = AttnC(q.data_ptr(), out.data_ptr(), DTYPE_CODES[dtype], heads, q_stride, out_stride,
              _ints(lens, batch, "lens", index), plan.max_len, window,
              dim ** -0.5 if scale is None else scale, None if lse is None else lse.data_ptr(),
              w_in, w_out, width)
    _call(lib().qg_paged_attn, index, cache._ref, _byref(a), plan.workspace_at,
          _raw_stream(index) if stream is None else stream.cuda_stream)
    return out if lse is None else (out, lse)


def evict(cache: PagedCache, lens: torch.Tensor, weight: torch.Tensor, budget: int, *, sink: int = 0,
          recent: int = 0, new_table: torch.Tensor | None = None, lens_out: torch.Tensor | None = None,
          weight_out: torch.Tensor | None = None, kept: torch.Tensor | None = None, stream=None):
    """qg_kv_evict: keep `budget` slots per kv head of every longer sequence -- the first `sink`,
    the last `recent`, and the heaviest between them by weight [sequences, kv heads, >= longest
    length].  Rows move to the front of the same pages, lens and weight are updated; or, with
    new_table [sequences, pages], to those pages, the new weights to weight_out (needed then; it
    may be weight) and lens left as it is.  Returns (kept [sequences, kv heads, budget], new lens)."""
    index, batch, kv = cache.index, cache.batch, cache.n_kv_heads
    if weight.dim() != 3:
        _fail("weight: [sequences, kv heads, slots] is needed")
    width = weight.shape[2]
    shape = (batch, kv, width)
    weight_at, lens_at = _floats(weight, shape, "weight", index), _ints(lens, batch, "lens", index)
    to, pages, step, elsewhere = None, 0, 0, new_table is not None
    if elsewhere:
        if (new_table.dtype is not _I32 or new_table.dim() != 2 or new_table.get_device() != index
                or new_table.shape[0] != batch):
            _fail("new_table: an int32 tensor [sequences, pages per sequence] is needed")
        pages = new_table.shape[1]
        step, one = new_table.stride()
        if one != 1 and pages > 1:
            _fail("new_table: a sequence's pages must be contiguous")
        to, step = new_table.data_ptr(), step if batch > 1 else pages
    if lens_out is None and elsewhere:
        lens_out = _like(lens, stream)
        lens_out_at = lens_out.data_ptr()
    elif lens_out is None or lens_out is lens:
        lens_out, lens_out_at = lens, lens_at
    else:
        lens_out_at = _ints(lens_out, batch, "lens_out", index)
    if weight_out is None and elsewhere:
        _fail("new_table needs weight_out: a tensor for the new weights, or weight itself")
    if weight_out is None or weight_out is weight:
        weight_out_at = weight_at
    else:
        weight_out_at = _floats(weight_out, shape, "weight_out", index)
    if kept is None:
        kept = _new_ints((batch, kv, budget), lens, stream)
        kept_at = kept.data_ptr()
    else:
        kept_at = _ints(kept, batch * kv * budget, "kept", index)
    e = EvictC(lens_at, lens_out_at, weight_at, weight_out_at, width, width, budget, sink, recent, kept_at,
               to, pages, step)
    _call(lib().qg_kv_evict, index, cache._ref, _byref(e),
          _raw_stream(index) if stream is None else stream.cuda_stream)
    return kept, lens_out
