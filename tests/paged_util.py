"""Paged caches for the tests: pools and page tables in any layout, their logical rows, and
the unit roundoffs that the tolerances are made of; the C-ABI's structures."""

import ctypes
from ctypes import c_float, c_int, c_uint32, c_uint64, c_void_p

import numpy as np
import torch

from qgemv_b200 import paged

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}  # half the least subnormal
INVALID_VALUE = 1  # cudaErrorInvalidValue


def make_cache(rng, batch, table_pages, page, heads, dim, dtype, order="hsd", spare=2, dev="cuda",
               pad=0):
    """A cache of random rows; `order` is the order of heads and places inside a page, `pad`
    unused values follow every row.  Pages are handed out in a random order."""
    n = batch * table_pages + spare
    g = torch.Generator(device=dev)
    g.manual_seed(int(rng.integers(1 << 31)))

    def pool():
        shape = (n, heads, page, dim + pad) if order == "hsd" else (n, page, heads, dim + pad)
        t = torch.empty(shape, dtype=dtype, device=dev).normal_(generator=g)
        t = t if order == "hsd" else t.permute(0, 2, 1, 3)
        return t[..., :dim]

    table = torch.from_numpy(rng.permutation(n)[: batch * table_pages].astype(np.int32))
    return paged.PagedCache(pool(), pool(), table.view(batch, table_pages).to(dev))


def row_index(cache, seq, slots):
    """(page, place) of slots of a sequence, as int64 tensors on the pool's device."""
    slots = torch.as_tensor(slots, dtype=torch.int64, device=cache.device)
    return cache.table[seq].long()[slots // cache.page_size], slots % cache.page_size


def logical(cache, pool, seq, n):
    """The first n slots of a sequence: [heads, n, dim] in float64 on the CPU."""
    page, place = row_index(cache, seq, torch.arange(n))
    return pool[page, :, place].double().cpu().transpose(0, 1)


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
