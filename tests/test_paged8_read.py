"""qg_kv_read8 (paged8.read): code times scale in fp32, rounded once to the type of the rows.  With
scales that are powers of two the product is exact, so the rows are equal to the rounding of the
exact value; with others within one fp32 rounding more."""

import ctypes

import numpy as np
import pytest
import torch

import qgemv_b200
from paged8_util import BAD_PAGES, codes, int32, logical, make_cache, offsets, pages_c, Read8C
from paged_util import DTYPES, INVALID_VALUE
from qgemv_b200 import ops, paged, paged8


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,dim,page,block,order,counts,starts", [
    (8, 128, 32, 32, "hsd", [1], [0]),
    (1, 16, 16, 16, "hsd", [40, 0, 3], [5, 1, 29]),     # the smallest row
    (3, 80, 48, 16, "shd", [0, 100, 1, 0, 37], [0, 44, 143, 9, 0]),
    (2, 256, 128, 128, "shd", [300], [84]),
    (4, 112, 96, 32, "hsd", [95, 96, 97], [1, 0, 95]),
    (1, 64, 64, 64, "hsd", [int(n) for n in np.arange(700) % 4], [int(n) for n in np.arange(700) % 60]),
])
def test_read(cuda, heads, dim, page, block, order, counts, starts, dtype):
    rng = np.random.default_rng(dim + page)
    longest = max(s + n for s, n in zip(starts, counts))
    c = make_cache(rng, len(counts), -(-longest // page), page, block, heads, dim, order, pad=16)
    codes(c.k)[0, :, :, 0] = 0x7F  # NaN
    rows = sum(counts) + 3
    k = torch.full((rows, heads, dim), 9.0, dtype=DTYPES[dtype], device="cuda")
    v = torch.full((rows, heads + 2, dim), 9.0, dtype=DTYPES[dtype], device="cuda")[:, 1: heads + 1]
    got = paged8.read(c, int32(starts), offsets(counts), rows, dtype=DTYPES[dtype], k_out=k, v_out=v)
    assert got[0].data_ptr() == k.data_ptr() and got[1].data_ptr() == v.data_ptr()
    row = 0
    for b, (s, n) in enumerate(zip(starts, counts)):
        for name, t in (("k", k), ("v", v)):
            want = logical(c, name, b, s + n)[:, s:].transpose(0, 1).to(DTYPES[dtype])
            assert torch.equal(t[row: row + n].cpu().nan_to_num(1e4), want.nan_to_num(1e4))
        row += n
    assert (k[row:] == 9).all() and (v[row:] == 9).all() and ops.get_error() == 0


@pytest.mark.gpu
def test_read_back_what_was_appended(cuda):
    """Through the cache and back: within half an e4m3 step of the block's values."""
    rng = np.random.default_rng(1)
    c = make_cache(rng, 2, 3, 64, 32, 2, 128)
    k, v = (torch.from_numpy(rng.standard_normal((200, 2, 128))).float().cuda() for _ in range(2))
    q = torch.empty(200, 0, 128, device="cuda")
    paged8.qk_norm_rope_append(c, q, k, v, None, int32([0] * 200), int32([150, 50]), offsets=offsets([150, 50]))
    got = paged8.read(c, int32([0, 0]), offsets([150, 50]), 200, dtype=torch.float32)
    for x, y in zip((k, v), got):
        assert ((x - y).abs() <= 2.0 ** -4 * x.abs() + 2.0 ** -16).all()  # scales are 2^-6 at most
    assert ops.get_error() == 0


@pytest.mark.gpu
def test_read_scales_that_are_no_powers(cuda):
    rng = np.random.default_rng(2)
    c = make_cache(rng, 1, 2, 32, 16, 2, 64)
    c.k_scale.mul_(1.37)
    k, _ = paged8.read(c, int32([0]), offsets([64]), 64, dtype=torch.float32)
    want = logical(c, "k", 0, 64).transpose(0, 1)
    assert ((k.double().cpu() - want).abs() <= 2.0 ** -24 * want.abs()).all()


@pytest.mark.gpu
def test_read_what_does_not_fit(cuda):
    """Slots outside the table and pages outside the pool give zero rows, and are reported."""
    rng = np.random.default_rng(3)
    c = make_cache(rng, 2, 2, 32, 16, 2, 64)
    ref, _ = paged8.read(c, int32([0, 0]), offsets([64, 64]), 128)
    for starts, zero in (([-3, 0], slice(0, 3)), ([10, 0], slice(54, 64)), ([0, 2 ** 31 - 40], slice(64, 128))):
        k, v = paged8.read(c, int32(starts), offsets([64, 64]), 128)
        assert (k[zero] == 0).all() and (v[zero] == 0).all() and ops.get_error() == paged.QG_ERR_PAGE
    for bad in (-1, c.num_pages):
        old = c.table[1, 1].clone()
        c.table[1, 1] = bad
        k, _ = paged8.read(c, int32([0, 0]), offsets([64, 64]), 128)
        assert torch.equal(k[:96], ref[:96]) and (k[96:] == 0).all() and ops.get_error() == paged.QG_ERR_PAGE
        c.table[1, 1] = old
    k, _ = paged8.read(c, int32([0, 0]), offsets([64, 65]), 128)  # more rows than the call has
    assert torch.equal(k, ref) and ops.get_error() == paged.QG_ERR_PAGE
    k, _ = paged8.read(c, int32([0, 0]), int32([-4, 64, 128]), 128)
    assert torch.equal(k[64:], ref[64:]) and ops.get_error() == paged.QG_ERR_PAGE
    assert paged8.read(c, int32([0, 0]), offsets([0, 0]), 0)[0].shape == (0, 2, 64) and ops.get_error() == 0


@pytest.mark.gpu
def test_read_offsets_past_32_bits_and_streams(cuda):
    heads, page, dim = 8, 128, 128
    n = 2 ** 32 // (heads * page * dim) + 3
    pool = torch.zeros(2, n, heads, page, dim, dtype=torch.uint8, device="cuda")
    pool[:, -2:] = torch.randint(0, 127, pool[:, -2:].shape, device="cuda").to(torch.uint8)
    scale = torch.ones(2, n, heads, 4, device="cuda")
    c = paged8.PagedCache8(*(p.view(torch.float8_e4m3fn) for p in pool), *scale, int32([[n - 1, n - 2]]))
    s = torch.cuda.Stream()
    starts, off = int32([100]), offsets([150])
    s.wait_stream(torch.cuda.current_stream())
    k, v = paged8.read(c, starts, off, 150, dtype=torch.bfloat16, stream=s)
    s.synchronize()
    for name, t in (("k", k), ("v", v)):
        assert torch.equal(t.double().cpu(), logical(c, name, 0, 250)[:, 100:].transpose(0, 1))
    rows = 2 ** 32 // (heads * dim * 2) + 10  # rows of more than 2^32 bytes
    out = torch.zeros(2, rows, heads, dim, dtype=torch.float16, device="cuda")
    off = int32([rows - 20])
    paged8.read(c, int32([3]), torch.cat([off, off + 20]), rows, k_out=out[0], v_out=out[1])
    for i, name in enumerate("kv"):
        assert torch.equal(out[i, -20:].double().cpu(), logical(c, name, 0, 23)[:, 3:].transpose(0, 1))
    assert torch.count_nonzero(out[:, : rows - 20]) == 0 and ops.get_error() == 0


@pytest.mark.gpu
def test_read_front_end_refuses(cuda):
    rng = np.random.default_rng(4)
    c = make_cache(rng, 2, 2, 32, 16, 2, 64)
    ok = dict(starts=int32([0, 0]), offsets=offsets([1, 1]), tokens=2)
    out = torch.empty(2, 2, 64, dtype=torch.float16, device="cuda")
    for b in (dict(starts=int32([0])), dict(starts=int32([0, 0]).long()), dict(offsets=int32([0, 1])), dict(tokens=-1),
              dict(dtype=torch.float64), dict(dtype=torch.float8_e4m3fn), dict(k_out=out[:1]), dict(v_out=out.float()),
              dict(v_out=out.cpu()), dict(offsets=offsets([1, 1]).cpu())):
        with pytest.raises(ValueError):
            paged8.read(c, **(ok | b))
    assert paged8.read(c, **ok)[0].shape == (2, 2, 64) and ops.get_error() == 0


def _args():
    return pages_c(), Read8C(64, 64, 5, 64, 64, 1, 128, 128)


@pytest.mark.parametrize("field,value", BAD_PAGES)
def test_read_refuses_bad_caches(field, value):
    c, r = _args()
    setattr(c, field, value)
    assert qgemv_b200.call("qg_kv_read8", ctypes.byref(c), ctypes.byref(r), None) == INVALID_VALUE


@pytest.mark.parametrize("field,value", [
    ("starts", None), ("offsets", None), ("tokens", 2 ** 31), ("k_out", None), ("k_out", 8), ("v_out", None),
    ("v_out", 72), ("dtype", 3), ("dtype", -1), ("k_stride", 132), ("v_stride", 4),
])
def test_read_refuses_bad_arguments(field, value):
    c, r = _args()
    setattr(r, field, value)
    assert qgemv_b200.call("qg_kv_read8", ctypes.byref(c), ctypes.byref(r), None) == INVALID_VALUE


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_read_rows_that_begin_on_16_bytes(cuda, dtype):
    """Outputs 16 bytes past a 32-byte boundary, or with such strides: the same bits, and nothing beside them."""
    rng = np.random.default_rng(8)
    c = make_cache(rng, 3, 4, 64, 32, 3, 80)
    starts, ends = int32([7, 0, 100]), offsets([90, 64, 33])
    dt = DTYPES[dtype]
    want = paged8.read(c, starts, ends, 190, dtype=dt)
    few = 16 // dt.itemsize
    for lead, tail in ((few, 0), (0, few), (few, few)):
        wide = [torch.full((190, 3 * 80 + lead + tail), 9.0, dtype=dt, device="cuda") for _ in range(2)]
        outs = [w[:, lead: lead + 240].unflatten(1, (3, 80)) for w in wide]
        paged8.read(c, starts, ends, 190, dtype=dt, k_out=outs[0], v_out=outs[1])
        for w, out, x in zip(wide, outs, want):
            assert torch.equal(out[:187], x[:187]) and (out[187:] == 9).all()
            assert (w[:, :lead] == 9).all() and (w[:, lead + 240:] == 9).all()
    assert ops.get_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("batch", [3, 300])
def test_read_reports_offsets_that_do_not_ascend(cuda, batch):
    """Wherever in the list they are: an offset below the one before it, below zero, or past the call's rows."""
    rng = np.random.default_rng(9)
    c = make_cache(rng, batch, 1, 32, 16, 1, 64)
    starts, good = int32([0] * batch), np.arange(batch + 1) * 4
    tokens = 4 * batch
    paged8.read(c, starts, int32(good.tolist()), tokens)
    assert ops.get_error() == 0
    for at, value in ((1, 9), (1, -1), (1, tokens + 1), (batch - 1, 2), (batch // 2 + 1, tokens + 5), (batch, 0),
                      (batch, tokens - 5), (batch, tokens + 1), (0, -1), (0, 5)):
        off = good.copy()
        off[at] = value
        for rows in (tokens, 3):  # also where the call has fewer CTAs than sequences
            paged8.read(c, starts, int32(off.tolist()), rows)
            assert ops.get_error() == paged.QG_ERR_PAGE, (at, value, rows)
