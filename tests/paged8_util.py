"""8-bit paged caches for the tests: pools, scales and tables in any layout, their rows in 64 bits,
e4m3 rounding, the C-ABI's structures."""

import ctypes
from ctypes import c_float, c_int, c_uint32, c_uint64, c_void_p

import numpy as np
import torch

from qgemv_b200 import paged8


def codes(t):
    """The bytes of a float8 tensor (views of any strides)."""
    return t.view(torch.uint8)


def values(t):
    return codes(t).contiguous().view(torch.float8_e4m3fn).double()


def e4m3(x):
    """Nearest e4m3 values of a float64 array, ties to even, past the range its end; NaN stays."""
    size = np.clip(np.nan_to_num(np.abs(x), nan=1.0), 2.0 ** -6, 448.0)
    step = np.exp2(np.floor(np.log2(size)) - 3)
    return np.clip(np.round(x / step) * step, -448, 448)


def make_cache(rng, batch, table_pages, page, block, heads, dim, order="hsd", spare=2, dev="cuda", pad=0,
               power=0):
    """A cache of random codes with scales 2^(power - 9) to 2^(power - 5); `order` is the order of heads and
    places inside a page, `pad` unused bytes follow every row.  Pages are handed out in a random order."""
    n = batch * table_pages + spare
    g = torch.Generator(device=dev)
    g.manual_seed(int(rng.integers(1 << 31)))

    def pool():
        shape = (n, heads, page, dim + pad) if order == "hsd" else (n, page, heads, dim + pad)
        t = torch.empty(shape, device=dev).normal_(generator=g).mul_(100).clamp_(-448, 448)
        t = t.to(torch.float8_e4m3fn)
        return codes(t if order == "hsd" else codes(t).permute(0, 2, 1, 3).view(torch.float8_e4m3fn))[..., :dim].view(
            torch.float8_e4m3fn)

    def scale():
        e = torch.randint(power - 9, power - 4, (n, heads, page // block), generator=g, device=dev)
        return torch.exp2(e.double()).float()

    table = torch.from_numpy(rng.permutation(n)[: batch * table_pages].astype(np.int32))
    return paged8.PagedCache8(pool(), pool(), scale(), scale(), table.view(batch, table_pages).to(dev))


def places(cache, seq, slots):
    """(page, place) of slots of a sequence."""
    slots = torch.as_tensor(slots, dtype=torch.int64)
    assert slots.numel() == 0 or 0 <= slots.min() <= slots.max() < cache.capacity  # on the host, before any lookup
    slots = slots.to(cache.device)
    return cache.table[seq].long()[slots // cache.page_size], slots % cache.page_size


def logical(cache, name, seq, n):
    """The first n slots of a sequence's keys or values: [heads, n, dim] in float64 on the CPU."""
    page, place = places(cache, seq, torch.arange(n))
    c = codes(getattr(cache, name))[page, :, place].view(torch.float8_e4m3fn).double()
    s = getattr(cache, name + "_scale")[page, :, place // cache.block].double()
    return (c * s[..., None]).cpu().transpose(0, 1)


def int32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def offsets(counts):
    return int32([0] + [int(n) for n in np.cumsum(counts)])


class KvPages8C(ctypes.Structure):
    _fields_ = [("k", c_void_p), ("v", c_void_p), ("k_scale", c_void_p), ("v_scale", c_void_p),
                ("num_pages", c_uint32), ("page_size", c_uint32), ("n_kv_heads", c_uint32),
                ("head_dim", c_uint32), ("block", c_uint32), ("page_stride", c_uint64), ("head_stride", c_uint64),
                ("slot_stride", c_uint64), ("scale_page_stride", c_uint64), ("scale_head_stride", c_uint64),
                ("table", c_void_p), ("batch", c_uint32), ("table_pages", c_uint32), ("table_stride", c_uint32)]


class Append8C(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("k", c_void_p), ("v", c_void_p), ("q_out", c_void_p),
                ("dtype", c_int), ("tokens", c_uint32), ("n_q_heads", c_uint32),
                ("q_stride", c_uint64), ("k_stride", c_uint64), ("v_stride", c_uint64),
                ("q_out_stride", c_uint64), ("q_norm", c_void_p), ("k_norm", c_void_p),
                ("eps", c_float), ("rope", c_void_p), ("rope_rows", c_uint32),
                ("rot_dim", c_uint32), ("pairs", c_int), ("positions", c_void_p),
                ("lens", c_void_p), ("offsets", c_void_p)]


class Read8C(ctypes.Structure):
    _fields_ = [("starts", c_void_p), ("offsets", c_void_p), ("tokens", c_uint32), ("k_out", c_void_p),
                ("v_out", c_void_p), ("dtype", c_int), ("k_stride", c_uint64), ("v_stride", c_uint64)]


class Attn8C(ctypes.Structure):
    _fields_ = [("q", c_void_p), ("out", c_void_p), ("dtype", c_int), ("tokens", c_uint32),
                ("n_q_heads", c_uint32), ("q_stride", c_uint64), ("out_stride", c_uint64),
                ("lens", c_void_p), ("offsets", c_void_p), ("window", c_uint32), ("sink", c_uint32),
                ("scale", c_float), ("lse", c_void_p)]


def pages_c():
    """A cache description that every entry point accepts (addresses that nothing is read from)."""
    return KvPages8C(64, 64, 64, 64, 4, 32, 2, 64, 16, 4096, 2048, 64, 4, 2, 64, 2, 2, 2)


BAD_PAGES = [("k", None), ("k", 8), ("v", None), ("v", 72), ("k_scale", None), ("k_scale", 66), ("v_scale", None),
             ("num_pages", 0), ("num_pages", 2 ** 31), ("page_size", 0), ("page_size", 24), ("n_kv_heads", 0),
             ("n_kv_heads", 32768), ("head_dim", 0), ("head_dim", 24), ("head_dim", 272), ("block", 0), ("block", 8),
             ("block", 24), ("block", 64), ("block", 256), ("page_stride", 4104), ("head_stride", 1032),
             ("slot_stride", 72), ("table", None), ("batch", 0), ("batch", 65536), ("table_pages", 0),
             ("table_stride", 1), ("table_pages", 2 ** 31 - 1)]
