"""qg_paged_attn8 (paged8.attend) against softmax(q K^T) V in 64 bits, row by row of the mask.

Tolerances.  A score of sizes |q| |k| scale = c is off by at most ds = 2^-20 c (queries carry 22 bits, or
24 below their row's largest value; fp32 accumulation over up to 256 products, truncating,
included).  A probability's relative error is then ds and 2^-17 for exp2, the running maximum and the
rounding of score plus log2 scale, together below 64 in size; its own split leaves 2^-20.  So
|out - want| <= (2 ds + 2^-16) max|v| + the rounding of the output type, and 2^-11 (fp16's unit
roundoff, times sum p |v| <= max|v|) more where 16-bit queries have more than 8 rows for a kv head;
lse within ds + 2^-19 |lse| + 2^-16."""

import ctypes

import numpy as np
import pytest
import torch

import qgemv_b200
from paged8_util import (Attn8C, BAD_PAGES, codes, int32, logical, make_cache, offsets, pages_c, places)
from paged_util import DTYPES, INVALID_VALUE, TINY, UNIT
from qgemv_b200 import ops, paged, paged8


def queries(rng, rows, heads, dim, dtype, scale=2.0):
    return torch.from_numpy(rng.standard_normal((rows, heads, dim)) * scale).to(dtype).cuda()


def mask(n, new, window, sink):
    slot, j = np.arange(n - new, n)[:, None], np.arange(n)[None]
    seen = j <= slot
    if window:
        seen &= (j > slot - window) | (j < sink)
    return torch.from_numpy(seen)


def check(cache, q, lens, counts, out, lse=None, window=0, sink=0, scale=None, tables=None):
    """Rows of all sequences, one after another; NaN where a seen code is one."""
    scale = q.shape[2] ** -0.5 if scale is None else scale
    kv, dim = cache.n_kv_heads, cache.head_dim
    group = q.shape[1] // kv
    qd, out = q.double().cpu(), out.double().cpu()
    coarse = 2.0 ** -11 if q.dtype != torch.float32 else 0.0
    row = 0
    for b, (n, new) in enumerate(zip(lens, counts)):
        rows = slice(row, row + new)
        row += new
        if n <= 0:
            assert (out[rows] == 0).all() and (lse is None or (lse[rows] == -np.inf).all())
            continue
        if new == 0:
            continue
        seen = mask(n, new, window, sink)
        k, v = (logical(cache, name, b, n) for name in "kv")
        ever = seen.any(0)
        k, v = (torch.where(ever[None, :, None], x, 0.0) for x in (k, v))
        for h in range(kv):
            mine = slice(h * group, (h + 1) * group)
            s = torch.einsum("tgd,jd->gtj", qd[rows, mine], k[h]) * scale
            s = s.masked_fill(~seen, -np.inf)
            want_lse = torch.logsumexp(s, -1).t()
            p = torch.softmax(s, -1)
            p = torch.where(seen, p, torch.zeros(()).double())
            clean = torch.nan_to_num(v[h], nan=0.0)
            want = torch.einsum("gtj,jd->tgd", p, clean)
            odd = torch.einsum("tj,jd->td", seen.double(), torch.isnan(v[h]).double()) > 0
            want[odd[:, None].expand(want.shape)] = np.nan
            got = out[rows, mine]
            assert torch.equal(torch.isnan(got), torch.isnan(want)), (b, h)
            ds = (qd[rows, mine].norm(dim=-1).max() * torch.nan_to_num(k[h]).norm(dim=-1).max()).item() * abs(scale) * 2.0 ** -20
            tol = (2 * ds + 2.0 ** -16 + coarse) * clean.abs().max() + UNIT[q.dtype] * 1.01 * want.abs() + TINY[q.dtype]
            fine = ~torch.isnan(want)
            assert ((got - want).abs() <= tol)[fine].all(), (b, h, (got - want)[fine].abs().max(), tol[fine].min())
            if lse is not None:
                err = (lse[rows, mine].double().cpu() - want_lse).abs()
                fine = torch.isfinite(want_lse)
                assert torch.equal(torch.isnan(err), torch.isnan(want_lse))
                assert (err <= ds + 2.0 ** -19 * want_lse.abs() + 2.0 ** -16)[fine].all(), (b, h, err[fine].max())


def poison(cache, lens):
    """NaN in every slot past its sequence's end, in every page of no sequence, and in the scales of
    blocks that hold nothing."""
    used = torch.zeros(cache.num_pages, cache.page_size, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        page, place = places(cache, b, torch.arange(max(n, 0)))
        used[page, place] = True
    blocks = used.unflatten(1, (-1, cache.block)).any(-1)
    for pool, scale in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        codes(pool).permute(0, 2, 1, 3)[~used] = 0x7F
        scale.permute(0, 2, 1)[~blocks] = float("nan")


SHAPES = [
    # q heads, kv heads, dim, page, block, order
    (64, 8, 128, 32, 32, "hsd"),
    (8, 8, 64, 48, 16, "shd"),      # one query head a kv head
    (3, 1, 80, 16, 16, "hsd"),
    (32, 2, 64, 64, 64, "hsd"),     # 16 heads
    (24, 2, 128, 96, 32, "shd"),    # 12 heads: tiles of two tokens
    (20, 1, 128, 128, 128, "hsd"),  # 20 heads over two tiles
    (40, 2, 256, 64, 32, "hsd"),
    (6, 2, 256, 48, 16, "shd"),
    (5, 5, 16, 32, 16, "hsd"),      # the smallest head
    (16, 4, 112, 128, 32, "shd"),
    (7, 1, 48, 16, 16, "shd"),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page,block,order", SHAPES)
def test_one_token_a_sequence(cuda, q_heads, kv_heads, dim, page, block, order, dtype):
    rng = np.random.default_rng(q_heads * 7 + dim)
    lens = [1, 16, 31, 32, 33, 0, 127, 128, 129, 700, -3, 255]
    c = make_cache(rng, len(lens), 704 // page + 1, page, block, kv_heads, dim, order)
    poison(c, lens)
    q = queries(rng, len(lens), q_heads, dim, DTYPES[dtype])
    plan = paged8.AttentionPlan8(c, q_heads)
    for window, sink in ((0, 0), (1, 0), (100, 0), (30, 5), (33, 200), (1, 1), (300, 17)):
        out, lse = paged8.attend(plan, q, int32(lens), window=window, sink=sink, return_lse=True)
        check(c, q, lens, [1] * len(lens), out, lse, window, sink)
        again = paged8.attend(plan, q, int32(lens), window=window, sink=sink)
        assert torch.equal(again, out)
    assert ops.get_error() == 0 and torch.count_nonzero(plan.workspace[:4096]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page,block,order", SHAPES)
def test_ragged_rows(cuda, q_heads, kv_heads, dim, page, block, order, dtype):
    """Prompts, chunks, drafted tokens, single tokens and nothing in one call, rows behind the last left
    alone; a call that is one long prompt."""
    rng = np.random.default_rng(q_heads * 7 + dim + 1)
    lens = [5, 700, 0, 64, 130, 1, 333, 0, 400]
    counts = [5, 3, 0, 64, 1, 1, 300, 2, 0]
    c = make_cache(rng, len(lens), 704 // page + 1, page, block, kv_heads, dim, order)
    poison(c, lens)
    rows = sum(counts)
    q = queries(rng, rows + 3, q_heads, dim, DTYPES[dtype])
    plan = paged8.AttentionPlan8(c, q_heads, max_tokens=rows + 3)
    for window, sink in ((0, 0), (1, 0), (100, 4), (20, 70), (250, 0)):
        out = torch.full_like(q, 3.0)
        lse = torch.full(q.shape[:2], 3.0, device="cuda")
        paged8.attend(plan, q, int32(lens), offsets=offsets(counts), window=window, sink=sink, out=out, lse=lse)
        check(c, q[:rows], lens, counts, out[:rows], lse[:rows], window, sink)
        assert (out[rows:] == 3).all() and (lse[rows:] == 3).all()
        again = torch.empty_like(q)
        paged8.attend(plan, q, int32(lens), offsets=offsets(counts), window=window, sink=sink, out=again)
        assert torch.equal(again[:rows], out[:rows])
    one = [0] * len(lens)
    one[1] = rows + 3
    out, lse = paged8.attend(plan, q, int32(lens), offsets=offsets(one), return_lse=True)
    check(c, q, lens, one, out, lse)
    assert ops.get_error() == 0 and torch.count_nonzero(plan.workspace[:4096]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page,block,order", SHAPES)
def test_drafted_tokens(cuda, q_heads, kv_heads, dim, page, block, order, dtype):
    """A few rows of every sequence."""
    rng = np.random.default_rng(q_heads * 7 + dim + 2)
    counts = [int(n) for n in rng.integers(0, 5 if q_heads // kv_heads < 12 else 3, 24)]
    lens = [n + int(m) for n, m in zip(counts, rng.integers(0, 600, 24))]
    c = make_cache(rng, 24, 640 // page + 1, page, block, kv_heads, dim, order)
    poison(c, lens)
    q = queries(rng, sum(counts), q_heads, dim, DTYPES[dtype])
    plan = paged8.AttentionPlan8(c, q_heads, max_tokens=sum(counts))
    for window, sink in ((0, 0), (2, 0), (100, 4), (64, 500)):
        out, lse = paged8.attend(plan, q, int32(lens), offsets=offsets(counts), window=window, sink=sink, return_lse=True)
        check(c, q, lens, counts, out, lse, window, sink)
    assert ops.get_error() == 0 and torch.count_nonzero(plan.workspace[:4096]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nan_reaches_only_rows_that_see_it(cuda, dim, dtype):
    """NaN codes at a later token's slot, before a window and between first tokens and window, in
    keys and in values; a NaN value is its column's alone."""
    rng = np.random.default_rng(dim)
    lens, counts = [300, 90, 200, 210], [40, 90, 3, 130]
    q = queries(rng, sum(counts), 8, dim, DTYPES[dtype])
    for name in "vk":
        c = make_cache(rng, 4, 320 // 32, 32, 16, 2, dim, power=1)
        poison(c, lens)
        pool = codes(getattr(c, name))
        for b, slot, head, col, value in ((0, 290, 0, 3, 0x7F), (0, 291, 1, dim - 1, 0xFF), (1, 40, 1, 7, 0xFF),
                                          (2, 5, 0, 0, 0x7F), (2, 60, 1, 9, 0x7F), (2, 198, 0, 11, 0x7F),
                                          (3, 0, 0, 1, 0x7F), (3, 100, 1, 2, 0x7F)):
            page, place = places(c, b, [slot])
            pool[page, head, place, col] = value
        plan = paged8.AttentionPlan8(c, 8, max_tokens=sum(counts))
        for window, sink in ((0, 0), (12, 0), (64, 2), (150, 9)):
            out, lse = paged8.attend(plan, q, int32(lens), offsets=offsets(counts), window=window, sink=sink,
                                     return_lse=True)
            check_nan = check if name == "v" else check_keys
            check_nan(c, q, lens, counts, out, lse, window, sink)
        one = paged8.AttentionPlan8(c, 8)
        out = paged8.attend(one, q[:4], int32(lens), window=12, sink=2)
        (check if name == "v" else check_keys)(c, q[:4], lens, [1] * 4, out, None, 12, 2)
    assert ops.get_error() == 0


def check_keys(cache, q, lens, counts, out, lse, window, sink):
    """As check, with NaN keys: a row that sees one is NaN, the others do not know of it."""
    row = 0
    for b, (n, new) in enumerate(zip(lens, counts)):
        seen = mask(n, new, window, sink)
        k = logical(cache, "k", b, n)
        for h in range(cache.n_kv_heads):
            odd = (seen & torch.isnan(k[h]).any(-1)).any(-1)
            group = q.shape[1] // cache.n_kv_heads
            got = out[row: row + new, h * group: (h + 1) * group].cpu()
            assert torch.isnan(got[odd]).all() and torch.isfinite(got[~odd]).all()
            if lse is not None:
                got = lse[row: row + new, h * group: (h + 1) * group].cpu()
                assert torch.isnan(got[odd]).all() and torch.isfinite(got[~odd]).all()
        row += new


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("power", [50, 0, -40])
def test_scales_of_all_sizes(cuda, power, dtype):
    """Blocks of values far apart in size, and of zeros with the least scale, in one row; keys likewise, with
    queries that make ordinary scores of them."""
    rng = np.random.default_rng(power % 100)
    lens, counts = [500, 77, 40], [30, 1, 40]
    c = make_cache(rng, 3, 16, 32, 16, 1, 128, power=power)
    wide = torch.randint(-20, 6, c.v_scale.shape, device="cuda")
    c.v_scale.copy_(torch.ldexp(c.v_scale, wide).clamp(2.0 ** -60, 2.0 ** 60))
    for slot in (0, 130, 136, 490):
        page, place = places(c, 0, [slot])
        codes(c.v)[page, :, place // 16 * 16: place // 16 * 16 + 16] = 0
        c.v_scale[page, :, place // 16] = 2.0 ** -60
    poison(c, lens)
    size = 2.0 ** -power if dtype == "f32" else 1.0  # fp16 queries cannot make up for such keys
    if dtype == "f16":
        c.k_scale.copy_(torch.ldexp(c.k_scale, torch.tensor(-power, device="cuda")))
        c.v_scale.copy_(torch.ldexp(c.v_scale, torch.tensor(-power, device="cuda")).clamp(2.0 ** -60, 2.0 ** 60))
    q = queries(rng, 71, 4, 128, DTYPES[dtype], 2.0 * size)
    plan = paged8.AttentionPlan8(c, 4, max_tokens=71)
    out, lse = paged8.attend(plan, q, int32(lens), offsets=offsets(counts), return_lse=True)
    check(c, q, lens, counts, out, lse)
    out, lse = paged8.attend(plan, q[:3], int32(lens), return_lse=True)
    check(c, q[:3], lens, [1] * 3, out, lse)
    assert ops.get_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_queries_of_all_sizes(cuda, dtype):
    """Rows of zeros, of tiny and of large values, scores that leave one slot all the weight."""
    rng = np.random.default_rng(3)
    lens, counts = [140, 70], [60, 70]
    c = make_cache(rng, 2, 5, 32, 32, 2, 64, power=1)
    q = queries(rng, 130, 4, 64, DTYPES[dtype])
    q[3] = 0
    q[5] *= 1e-4
    q[7] *= 300.0
    q[9, :, 1:] = 0
    q[11] *= -1
    plan = paged8.AttentionPlan8(c, 4, max_tokens=130)
    for scale in (0.125, -0.5, 0.0, 3.0):
        out, lse = paged8.attend(plan, q, int32(lens), offsets=offsets(counts), return_lse=True, scale=scale)
        check(c, q, lens, counts, out, lse, scale=scale)
    assert ops.get_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_long_and_many(cuda, dtype):
    """A lone long sequence (records joined in groups), more sequences than a CTA has threads, ragged and not."""
    rng = np.random.default_rng(4)
    c = make_cache(rng, 1, 70000 // 64 + 1, 64, 64, 1, 64)
    q = queries(rng, 3, 2, 64, DTYPES[dtype])
    plan = paged8.AttentionPlan8(c, 2, max_tokens=3)
    for counts in ([1], [3]):
        out, lse = paged8.attend(plan, q[: counts[0]], int32([69990]), offsets=offsets(counts), return_lse=True)
        check(c, q[: counts[0]], [69990], counts, out, lse)
    out = paged8.attend(plan, q[:1], int32([69990]), window=60000, sink=9)
    check(c, q[:1], [69990], [1], out, None, 60000, 9)
    lens = [int(n) for n in rng.integers(0, 90, 1500)]
    counts = [min(n, int(m)) for n, m in zip(lens, rng.integers(0, 4, 1500))]
    c = make_cache(rng, 1500, 3, 32, 16, 2, 64)
    q = queries(rng, max(1500, sum(counts)), 6, 64, DTYPES[dtype])
    plan = paged8.AttentionPlan8(c, 6, max_tokens=len(q))
    out, lse = paged8.attend(plan, q[: sum(counts)], int32(lens), offsets=offsets(counts), return_lse=True)
    check(c, q[: sum(counts)], lens, counts, out, lse)
    out = paged8.attend(plan, q[:1500], int32(lens), window=40, sink=3)
    check(c, q[:1500], lens, [1] * 1500, out, None, 40, 3)
    # many sequences of many rows each: more tiles than SMs, some cut between them
    counts = [int(n) for n in rng.integers(0, 130, 120)]
    lens = [n + int(m) for n, m in zip(counts, rng.integers(0, 500, 120))]
    for dim, heads, kv in ((128, 8, 2), (48, 3, 1)):
        c = make_cache(rng, 120, 20, 32, 16, kv, dim)
        q = queries(rng, sum(counts), heads, dim, DTYPES[dtype])
        plan = paged8.AttentionPlan8(c, heads, max_tokens=len(q))
        for window, sink in ((0, 0), (90, 7)):
            out, lse = paged8.attend(plan, q, int32(lens), offsets=offsets(counts), window=window, sink=sink, return_lse=True)
            check(c, q, lens, counts, out, lse, window, sink)
    assert ops.get_error() == 0


@pytest.mark.gpu
def test_strides_streams_outputs_and_plans_at_once(cuda):
    rng = np.random.default_rng(5)
    c = make_cache(rng, 3, 3, 32, 16, 2, 64, pad=16)
    wide = queries(rng, 40, 10, 64, torch.float16)
    q, out = wide[:, 2:6], torch.full((40, 12, 64), 5.0, dtype=torch.float16, device="cuda")
    lens, counts = [64, 1, 33], [30, 1, 9]
    s = torch.cuda.Stream()
    plans = [paged8.AttentionPlan8(c, 4, max_tokens=40) for _ in range(2)]
    args = int32(lens), offsets(counts)
    ref = paged8.attend(plans[0], q, args[0], offsets=args[1])
    s.wait_stream(torch.cuda.current_stream())
    for _ in range(20):  # calls that overlap, a plan each
        paged8.attend(plans[0], q, args[0], offsets=args[1], out=out[:, 4:8], stream=s)
        here = paged8.attend(plans[1], q, args[0], offsets=args[1])
    s.synchronize()
    check(c, q, lens, counts, out[:, 4:8])
    assert torch.equal(here, ref) and torch.equal(out[:, 4:8], ref)
    assert (out[:, :4] == 5).all() and (out[:, 8:] == 5).all() and ops.get_error() == 0


@pytest.mark.gpu
def test_lengths_offsets_and_pages_that_do_not_fit(cuda):
    rng = np.random.default_rng(6)
    c = make_cache(rng, 3, 3, 32, 16, 2, 64)
    q = queries(rng, 30, 4, 64, torch.float16)
    plan = paged8.AttentionPlan8(c, 4, max_tokens=30)
    ref = paged8.attend(plan, q[:3], int32([96, 0, 33]))
    got = paged8.attend(plan, q[:3], int32([97, -3, 33]))  # one past the table: cut; negative: none
    assert torch.equal(got, ref) and ops.get_error() == paged.QG_ERR_PAGE
    out = torch.zeros_like(q)
    paged8.attend(plan, q, int32([96, 50, 33]), offsets=offsets([5, 5, 5]), out=out)
    for lens, off, dead in (([97, 50, 33], [0, 5, 10, 15], slice(0, 5)), ([96, 4, 33], [0, 5, 10, 15], slice(5, 10))):
        got = torch.full_like(q, 9.0)
        paged8.attend(plan, q, int32(lens), offsets=int32(off), out=got)  # rows that do not fit: zeros
        live = [i for i in range(15) if not dead.start <= i < dead.stop]
        assert torch.equal(got[live], out[live]) and (got[dead] == 0).all() and (got[15:] == 9).all()
        assert ops.get_error() == paged.QG_ERR_PAGE
    for off in ([0, 40, 40, 40], [9, 3, 10, 15], [-2, 5, 10, 15], [0, 30, 0, 30]):
        paged8.attend(plan, q, int32([96, 96, 96]), offsets=int32(off), out=got)  # never outside
        assert ops.get_error() == paged.QG_ERR_PAGE
    torch.cuda.synchronize()
    c.table[1, 2:] = torch.tensor([-1], dtype=torch.int32)  # past the length: not looked at
    paged8.attend(plan, q, int32([96, 50, 33]), offsets=offsets([5, 5, 5]), out=got)
    assert torch.equal(got[:15], out[:15]) and ops.get_error() == 0
    for bad in (-1, c.num_pages):
        c.table[0, 1] = bad
        paged8.attend(plan, q, int32([96, 50, 33]), offsets=offsets([5, 5, 5]), out=got)
        assert torch.equal(got[5:15], out[5:15]) and torch.isfinite(got[:5]).all()
        assert ops.get_error() == paged.QG_ERR_PAGE


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 40])
def test_offsets_past_32_bits(cuda, rows):
    page, heads, dim = 128, 8, 128
    n = 2 ** 32 // (page * heads * dim) + 3
    pool = torch.zeros(2, n, heads, page, dim, dtype=torch.uint8, device="cuda")
    pool[:, -2:] = torch.randint(0, 100, pool[:, -2:].shape, device="cuda").to(torch.uint8)
    scale = torch.full((2, n, heads, 4), 2.0 ** -3, device="cuda")
    c = paged8.PagedCache8(*(p.view(torch.float8_e4m3fn) for p in pool), *scale, int32([[n - 1, n - 2]]))
    rng = np.random.default_rng(8)
    q = queries(rng, rows, 16, dim, torch.float16)
    plan = paged8.AttentionPlan8(c, 16, max_tokens=rows)
    out = paged8.attend(plan, q, int32([250]), offsets=None if rows == 1 else offsets([rows]))
    check(c, q, [250], [rows], out)


@pytest.mark.gpu
def test_a_captured_call_follows_lengths_and_offsets(cuda):
    rng = np.random.default_rng(9)
    c = make_cache(rng, 2, 20, 32, 32, 2, 128)
    q = queries(rng, 60, 16, 128, torch.bfloat16)
    plans = [paged8.AttentionPlan8(c, 16, max_tokens=60) for _ in range(2)]
    lens, off, out, one = int32([1, 0]), offsets([1, 0]), torch.empty_like(q), torch.empty_like(q[:2])
    paged8.attend(plans[0], q, lens, offsets=off, out=out)
    paged8.attend(plans[1], q[:2], lens, out=one)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged8.attend(plans[0], q, lens, offsets=off, out=out, window=200, sink=3)
        paged8.attend(plans[1], q[:2], lens, out=one)
    for n, new in (([1, 0], [1, 0]), ([300, 77], [30, 30]), ([640, 2], [58, 2]), ([0, 640], [0, 60]), ([5, 5], [0, 0])):
        lens.copy_(int32(n))
        off.copy_(offsets(new))
        graph.replay()
        check(c, q[: sum(new)], n, new, out[: sum(new)], None, 200, 3)
        check(c, q[:2], n, [1, 1], one)
    assert ops.get_error() == 0


@pytest.mark.gpu
def test_front_end_refuses(cuda):
    rng = np.random.default_rng(16)
    c = make_cache(rng, 2, 2, 32, 16, 2, 64)
    q, plan, lens = queries(rng, 2, 4, 64, torch.float16), paged8.AttentionPlan8(c, 4, max_tokens=5), int32([3, 4])
    for bad in (dict(window=-1), dict(sink=-1), dict(out=q[:1]), dict(out=q.float()), dict(lse=q), dict(offsets=lens),
                dict(offsets=offsets([1, 1]).long()), dict(offsets=offsets([1, 1]).cpu())):
        with pytest.raises(ValueError):
            paged8.attend(plan, q, lens, **bad)
    for bad_q in (q[0], q.double(), q.cpu(), q.transpose(0, 1), q.repeat(1, 1, 2)[..., ::2], q.repeat(2, 1, 1), q[:, :3],
                  q.repeat(3, 1, 1)):
        with pytest.raises(ValueError):
            paged8.attend(plan, bad_q, lens)
    with pytest.raises(ValueError):
        paged8.attend(plan, q.repeat(3, 1, 1), lens, offsets=offsets([2, 4]))  # more rows than the plan's
    for bad_lens in (lens.long(), lens.cpu(), lens[:1]):
        with pytest.raises(ValueError):
            paged8.attend(plan, q, bad_lens)
    for heads in (0, 3, 65536):
        with pytest.raises(qgemv_b200.CudaError):
            paged8.AttentionPlan8(c, heads)
    with pytest.raises(AttributeError):
        plan.workspace = lens
    assert paged8.attend(plan, q[:0], lens, offsets=offsets([0, 0])).shape == (0, 4, 64)
    assert paged8.attend(plan, q, lens).shape == (2, 4, 64) and ops.get_error() == 0


def _args():
    return pages_c(), Attn8C(64, 64, 1, 2, 4, 256, 256, 64, None, 0, 0, 1.0, None)


@pytest.mark.parametrize("field,value", BAD_PAGES + [("head_stride", 1040), ("slot_stride", 48), ("page_stride", 5120)])
def test_attend_refuses_bad_caches(field, value):
    c, a = _args()
    setattr(c, field, value)
    assert qgemv_b200.call("qg_paged_attn8", ctypes.byref(c), ctypes.byref(a), 256, None) == INVALID_VALUE


@pytest.mark.parametrize("field,value", [
    ("q", None), ("q", 8), ("out", None), ("out", 24), ("dtype", -1), ("dtype", 3), ("tokens", 2 ** 31), ("tokens", 3),
    ("n_q_heads", 0), ("n_q_heads", 3), ("n_q_heads", 65536), ("q_stride", 4), ("out_stride", 260), ("lens", None),
])
def test_attend_refuses_bad_arguments(field, value):
    c, a = _args()
    setattr(a, field, value)
    assert qgemv_b200.call("qg_paged_attn8", ctypes.byref(c), ctypes.byref(a), 256, None) == INVALID_VALUE


def test_attend_refuses_bad_workspaces():
    c, a = _args()
    n = ctypes.c_size_t(0)
    for ws in (None, 128):
        assert qgemv_b200.call("qg_paged_attn8", ctypes.byref(c), ctypes.byref(a), ws, None) == INVALID_VALUE
    size = ("qg_paged_attn8_workspace_bytes", ctypes.byref(c))
    assert qgemv_b200.call(*size, 4, 2, ctypes.byref(n)) == 0 and n.value >= 4096
    few = n.value
    assert qgemv_b200.call(*size, 4, 4000, ctypes.byref(n)) == 0 and n.value >= few + 999 * 24 - 3 * 255  # three parts in whole 256 bytes
    assert qgemv_b200.call(*size, 3, 2, ctypes.byref(n)) == INVALID_VALUE
    assert qgemv_b200.call(*size, 4, 2 ** 31, ctypes.byref(n)) == INVALID_VALUE
    assert qgemv_b200.call(*size, 4, 2, None) == INVALID_VALUE
    a.tokens = 0
    assert qgemv_b200.call("qg_paged_attn8", ctypes.byref(c), ctypes.byref(a), 256, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])  # fp16 does not hold such values
@pytest.mark.parametrize("dim,group,rows", [(64, 2, 0), (128, 8, 0), (64, 2, 7), (128, 4, 5), (256, 1, 3), (64, 2, 30), (128, 8, 9)])
def test_values_at_both_ends_of_the_scales(cuda, dim, group, rows, dtype):
    """One block of the largest scale among 65520 slots of the least one, zeros and others: slots that weigh
    2^-12 to 2^-40 of one of the block's add up to a part of the softmax's sum, wherever the block lies.
    `rows` 0 is a call without offsets."""
    rng = np.random.default_rng(dim + group + rows)
    n, block, new = 65536, 16, max(rows, 1)
    table = int32([rng.permutation(n // 64).tolist()])
    code = lambda x: x.to(torch.float8_e4m3fn)  # noqa: E731
    scale = torch.full((2, n // 64, 1, 4), 1.0, device="cuda")
    scale[1] = 2.0 ** -60
    keys = torch.zeros(n // 64, 1, 64, dim, device="cuda")
    keys[..., 1] = torch.randint(-2, 3, keys.shape[:-1], device="cuda")
    for first in (0, n // 2, n - 64):
        page = int(table[0, first // 64])
        for small in (0.0, 50.0):
            k, s = keys.clone(), scale.clone()
            v = torch.randn(keys.shape, device="cuda") * small
            k[page, 0, :block, 0], s[1, page, 0, 0] = 16.0, 2.0 ** 60
            v[page, 0, :block] = torch.randn(block, dim, device="cuda") * 100
            c = paged8.PagedCache8(code(k), code(v.clamp(-448, 448)), *s, table)
            plan = paged8.AttentionPlan8(c, group, max_tokens=new)
            for powers in (0, 12, 18, 23, 40):
                q = torch.zeros(new, group, dim, dtype=DTYPES[dtype], device="cuda")
                q[..., 0] = powers * np.log(2) * dim ** 0.5 / 16
                q[..., 1] = torch.from_numpy(rng.standard_normal((new, group)))
                off = offsets([rows]) if rows else None
                out, lse = paged8.attend(plan, q, int32([n]), offsets=off, return_lse=True)
                check(c, q, [n], [new], out, lse)
    assert ops.get_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_few_rows_keep_22_bits(cuda, dim, dtype):
    """Calls of at most 8 rows for a kv head, with and without offsets: two slots whose values cancel but for the
    difference of their probabilities, which fp16 probabilities would round to 2^-12 of the values.  The head's
    bound without its fp16 term."""
    rng = np.random.default_rng(dim)
    cache_rng = np.random.default_rng(dim)
    for group, seqs, ragged in ((1, 40, False), (8, 9, False), (5, 3, False), (1, 1, True), (1, 8, True), (4, 2, True), (8, 1, True)):
        c = make_cache(cache_rng, seqs, 1, 32, 16, 2, dim, power=9)
        c.k_scale.fill_(2.0 ** -6)
        c.v_scale.fill_(1.0)
        page = c.table[:, 0].long()
        v = torch.randint(100, 400, (seqs, 2, dim), device="cuda").float().to(torch.float8_e4m3fn)
        codes(c.v)[page, :, 0], codes(c.v)[page, :, 1] = codes(v), codes(v) ^ 0x80
        q = queries(rng, seqs, 2 * group, dim, DTYPES[dtype], 0.5)
        plan = paged8.AttentionPlan8(c, 2 * group, max_tokens=seqs)
        out = paged8.attend(plan, q, int32([2] * seqs), offsets=offsets([1] * seqs) if ragged else None)
        for b in range(seqs):
            k, v = (logical(c, name, b, 2) for name in "kv")
            qd = q[b].double().cpu().view(2, group, dim)
            p = torch.softmax(torch.einsum("hgd,hjd->hgj", qd, k) * dim ** -0.5, -1)
            want = torch.einsum("hgj,hjd->hgd", p, v)
            ds = (qd.norm(dim=-1).max() * k.norm(dim=-1).max()).item() * dim ** -0.5 * 2.0 ** -20
            tol = (2 * ds + 2.0 ** -16) * v.abs().max() + UNIT[q.dtype] * 1.01 * want.abs() + TINY[q.dtype]
            off = (out[b].double().cpu().view(2, group, dim) - want).abs()
            assert (off <= tol).all(), (group, seqs, ragged, b, (off / tol).max())
    assert ops.get_error() == 0
