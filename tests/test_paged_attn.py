"""qg_paged_attn (paged.attend) against softmax(q K^T) V in 64 bits.

Tolerances.  q is split into 16-bit terms of at least 22 (fp16), 16 (bf16, exact for bf16 q)
or 24 bits (fp32 q over bf16), so a score of |q| |k| scale = c differs by at most
2^-20 c (fp32 accumulation over up to 256 products, truncating, included); ds below is that
bound in natural units.  A probability's relative error is then ds + 2^-19 (exp2, running
maximum), and in P V the probabilities' own split adds 2^-20 (fp16) or 2^-15 (bf16).  So
|out - want| <= (2 ds + 2^-18 + split) max|v| + the rounding of the output type;
lse within ds + 2^-19 |lse| + 2^-18; weights within (ds + 2^-18) of a slot's weight, for each
of the heads, plus fp32 sums."""

import ctypes

import numpy as np
import pytest
import torch

import qgemv_b200
from paged_util import AttnC, DTYPES, INVALID_VALUE, KvPagesC, logical, make_cache, row_index, TINY, UNIT
from qgemv_b200 import ops, paged


def formula(cache, q, lens, window, scale):
    """out, lse and every slot's summed shares, and (max |v|, the bound ds) per sequence."""
    batch, heads, dim = q.shape
    group = heads // cache.n_kv_heads
    out, lse = torch.zeros(batch, heads, dim).double(), torch.full((batch, heads), -np.inf).double()
    shares, size = [], []
    qd = q.double().cpu()
    for b, n in enumerate(lens):
        first = max(0, n - window) if window else 0
        share = torch.zeros(cache.n_kv_heads, n).double()
        top_v, ds = 0.0, 0.0
        if n > 0:
            k, v = (logical(cache, p, b, n)[:, first:] for p in (cache.k, cache.v))
            s = torch.matmul(qd[b].view(cache.n_kv_heads, group, dim), k.transpose(1, 2)) * scale
            lse[b] = torch.logsumexp(s, -1).view(-1)
            p = torch.softmax(s, -1)
            out[b] = torch.matmul(p, v).reshape(heads, dim)
            share[:, first:] = p.sum(1)
            top_v = v.abs().max().item()
            ds = (qd[b].norm(dim=-1).max() * k.norm(dim=-1).max()).item() * abs(scale) * 2.0 ** -20
        shares.append(share)
        size.append((top_v, ds))
    return out, lse, shares, size


def check(cache, q, lens, out, lse=None, window=0, scale=None, weight=None, before=None):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    want, want_lse, shares, size = formula(cache, q, lens, window, scale)
    out = out.double().cpu()
    coarse = 2.0 ** -15 if cache.dtype == torch.bfloat16 and q.dtype != torch.float32 else 2.0 ** -20
    group = q.shape[1] // cache.n_kv_heads
    for b, n in enumerate(lens):
        top_v, ds = size[b]
        tol = (2 * ds + 2.0 ** -18 + coarse) * top_v + UNIT[q.dtype] * 1.01 * want[b].abs() + TINY[q.dtype]
        assert ((out[b] - want[b]).abs() <= tol).all(), (b, n, (out[b] - want[b]).abs().max())
        if lse is not None and n == 0:
            assert (lse[b] == -np.inf).all()
        elif lse is not None:
            err = (lse[b].double().cpu() - want_lse[b]).abs()
            assert (err <= ds + 2.0 ** -19 * want_lse[b].abs() + 2.0 ** -18).all(), (b, err.max())
        if weight is not None:
            got, old = weight[b].double().cpu(), before[b].double().cpu()
            tol = (ds + 2.0 ** -18) * shares[b] + 2.0 ** -22 * group * (shares[b] + old[:, :n])
            assert ((got[:, :n] - old[:, :n] - shares[b]).abs() <= tol).all()
            assert torch.equal(got[:, n:], old[:, n:])


def poison(cache, lens, value):
    """Every slot past its sequence's end, and every page of no sequence."""
    used = torch.zeros(cache.num_pages, cache.page_size, dtype=torch.bool, device="cuda")
    for b, n in enumerate(lens):
        page, place = row_index(cache, b, torch.arange(n))
        used[page, place] = True
    for pool in (cache.k, cache.v):
        pool.permute(0, 2, 1, 3)[~used] = value


def queries(rng, batch, heads, dim, dtype, scale=2.0):
    return torch.from_numpy(rng.standard_normal((batch, heads, dim)) * scale).to(dtype).cuda()


def int32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


CASES = [
    # q heads, kv heads, dim, page, order, lengths
    (64, 8, 128, 16, "hsd", [1]),
    (64, 8, 128, 16, "hsd", [16, 17, 63, 64, 65, 0, 511]),
    (8, 8, 64, 24, "shd", [100, 1, 0, 333]),            # one query head a kv head
    (3, 1, 80, 7, "hsd", [5, 700]),                     # dims past 80 are padding
    (32, 2, 64, 1, "hsd", [130, 31]),                   # 16 heads: two tiles of 8 together
    (24, 2, 128, 100, "shd", [257, 999, 48]),           # 12 heads over two tiles
    (20, 1, 128, 32, "hsd", [1500]),                    # 20 heads: two passes
    (40, 2, 256, 64, "hsd", [129, 640]),                # 20 heads of 256: three passes
    (6, 2, 256, 48, "shd", [77, 0]),
    (5, 5, 8, 3, "hsd", [40, 2, 9]),                    # the smallest head
    (16, 4, 112, 16, "shd", [64] * 9),
]


@pytest.mark.gpu
@pytest.mark.parametrize("cache_type,q_type", [("f16", "f32"), ("f16", "f16"), ("bf16", "bf16"),
                                               ("bf16", "f32"), ("bf16", "f16"), ("f16", "bf16")])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page,order,lens", CASES)
def test_attend_matches_formula(cuda, cache_type, q_type, q_heads, kv_heads, dim, page, order, lens):
    rng = np.random.default_rng(q_heads * 7 + dim + len(lens))
    pages = -(-max(lens) // page) + 1
    c = make_cache(rng, len(lens), pages, page, kv_heads, dim, DTYPES[cache_type], order)
    poison(c, lens, float("nan"))
    q = queries(rng, len(lens), q_heads, dim, DTYPES[q_type])
    plan = paged.AttentionPlan(c, q_heads, weights=True)
    before = torch.rand(len(lens), kv_heads, plan.max_len, device="cuda")
    weight = before.clone()
    out, lse = paged.attend(plan, q, int32(lens), return_lse=True)
    check(c, q, lens, out, lse)
    again, lse2 = paged.attend(plan, q, int32(lens), return_lse=True, weight_in=weight, weight_out=weight)
    assert torch.equal(again, out) and torch.equal(lse, lse2)
    check(c, q, lens, again, lse2, weight=weight, before=before)
    assert ops.get_error() == 0
    assert torch.count_nonzero(plan.workspace[:4096]) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 15, 64, 100, 5000])
@pytest.mark.parametrize("page", [16, 23])
def test_attend_window(cuda, window, page):
    """Only the last `window` slots are seen, wherever they start; unseen slots keep their weight."""
    rng = np.random.default_rng(window + page)
    lens = [0, 1, 99, 100, 101, 640, 1013]
    c = make_cache(rng, len(lens), 1100 // page + 1, page, 2, 64, torch.float16)
    poison(c, lens, float("inf"))
    for b, n in enumerate(lens):  # nor are the slots before the window ever numbers
        page_ids, place = row_index(c, b, torch.arange(max(0, n - window)))
        c.v[page_ids, :, place] = float("nan")
    q = queries(rng, len(lens), 8, 64, torch.float32)
    plan = paged.AttentionPlan(c, 8, weights=True)
    before = torch.rand(len(lens), 2, plan.max_len + 5, device="cuda")
    weight = torch.full_like(before, 7.0)
    weight_in = before.clone()
    out, lse = paged.attend(plan, q, int32(lens), window=window, return_lse=True, weight_in=weight_in,
                            weight_out=weight)
    for b, n in enumerate(lens):
        assert (weight[b, :, n:] == 7.0).all()  # slots past the length are left alone
        weight[b, :, n:] = before[b, :, n:]
    check(c, q, lens, out, lse, window=window, weight=weight, before=before)
    assert torch.equal(weight_in, before) and ops.get_error() == 0


@pytest.mark.gpu
def test_attend_long_sequences_and_many_of_them(cuda):
    """Work split over every SM: one long sequence of few heads, and more sequences than one
    scan of the lengths takes, most of them short."""
    rng = np.random.default_rng(3)
    c = make_cache(rng, 1, 520, 64, 2, 128, torch.float16)
    q = queries(rng, 1, 16, 128, torch.float32)
    out, lse = paged.attend(paged.AttentionPlan(c, 16), q, int32([33201]), return_lse=True)
    check(c, q, [33201], out, lse)
    lens = [int(n) for n in rng.integers(0, 80, 300)]
    lens[137], lens[299] = 3001, 900
    c = make_cache(rng, 300, 95, 32, 2, 64, torch.bfloat16, "shd")
    poison(c, lens, float("nan"))
    q = queries(rng, 300, 4, 64, torch.bfloat16)
    out, lse = paged.attend(paged.AttentionPlan(c, 4), q, int32(lens), return_lse=True)
    check(c, q, lens, out, lse)
    assert ops.get_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("q_type,cache_type", [("f16", "f16"), ("bf16", "bf16"), ("f32", "bf16")])
@pytest.mark.parametrize("q_heads,kv_heads,dim,page,longest,window", [
    (4, 2, 128, 16, 64, 0),   # every warp with whole segments, more of them than warps
    (16, 2, 112, 5, 31, 0),
    (3, 3, 64, 24, 65, 40),   # three tiles, the window cutting into the first
    (8, 1, 80, 32, 1, 0),
])
def test_attend_many_short_sequences(cuda, q_type, cache_type, q_heads, kv_heads, dim, page, longest, window):
    rng = np.random.default_rng(dim + longest)
    batch = 700
    lens = [int(n) for n in rng.integers(0, longest + 1, batch)]
    lens[0], lens[1], lens[-1] = longest, 0, longest
    c = make_cache(rng, batch, longest // page + 1, page, kv_heads, dim, DTYPES[cache_type])
    poison(c, lens, float("nan"))
    q = queries(rng, batch, q_heads, dim, DTYPES[q_type])
    plan = paged.AttentionPlan(c, q_heads, weights=True)
    before = torch.rand(batch, kv_heads, plan.max_len, device="cuda")
    weight = before.clone()
    out, lse = paged.attend(plan, q, int32(lens), window=window, return_lse=True, weight_in=weight, weight_out=weight)
    check(c, q, lens, out, lse, window=window, weight=weight, before=before)
    lens = [longest] * batch  # as long as the pages reach: the same bits twice
    c2 = make_cache(rng, batch, longest // page + 1, page, kv_heads, dim, DTYPES[cache_type], "shd")
    plan = paged.AttentionPlan(c2, q_heads)
    out = paged.attend(plan, q, int32(lens), window=window)
    check(c2, q, lens, out, window=window)
    assert torch.equal(out, paged.attend(plan, q, int32(lens), window=window)) and ops.get_error() == 0


@pytest.mark.gpu
def test_attend_equal_scores_over_a_long_context(cuda):
    """Every probability alike and tiny, next to one that dominates: their sum must not drown
    in the 16-bit split of the probabilities."""
    rng = np.random.default_rng(4)
    n = 50000
    c = make_cache(rng, 1, n // 64 + 1, 64, 1, 64, torch.float16)
    c.k.zero_()
    c.v.fill_(1.0)
    page, place = row_index(c, 0, [777])
    c.k[page, :, place, 0] = 8.0
    c.v[page, :, place] = 0.0
    q = torch.zeros(1, 8, 64, device="cuda")
    q[0, :, 0] = torch.linspace(0, 2.2, 8, device="cuda")  # the one slot's share: none to nearly all
    out, lse = paged.attend(paged.AttentionPlan(c, 8), q, int32([n]), scale=1.0, return_lse=True)
    check(c, q, [n], out, lse, scale=1.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attend_small_large_and_infinite_values(cuda, dtype):
    """Queries far outside fp16's range keep their precision; a score of minus infinity in
    every slot leaves an empty row; a NaN stays in its own row."""
    rng = np.random.default_rng(5)
    c = make_cache(rng, 3, 10, 16, 1, 64, DTYPES[dtype])
    plan = paged.AttentionPlan(c, 4)
    for size in (1e-30, 1e30):
        q = queries(rng, 3, 4, 64, torch.float32) * size
        lens = [150, 3, 31]
        out, lse = paged.attend(plan, q, int32(lens), scale=0.2 / size, return_lse=True)
        check(c, q, lens, out, lse, scale=0.2 / size)
    page, place = row_index(c, 0, torch.arange(160))
    c.k[page, :, place] = 0
    c.k[page, :, place, 0] = float("inf")
    q = torch.zeros(3, 4, 64, device="cuda")
    q[0] = 1.0
    q[0, :, 0] = -1.0
    q[2, 1, 5] = float("nan")
    out, lse = paged.attend(plan, q, int32([150, 0, 31]), return_lse=True)
    assert torch.count_nonzero(out[:2]) == 0 and (lse[:2] == -np.inf).all()
    assert torch.isnan(out[2, 1]).all() and torch.isfinite(out[2, [0, 2, 3]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_attend_queries_near_the_largest_fp32(cuda, dtype):
    rng = np.random.default_rng(15)
    c = make_cache(rng, 2, 10, 16, 2, 128, DTYPES[dtype])
    q = queries(rng, 2, 4, 128, torch.float32) * 2e37  # up to about 2^126
    out, lse = paged.attend(paged.AttentionPlan(c, 4), q, int32([160, 33]), scale=4e-39, return_lse=True)
    assert torch.isfinite(out).all()
    check(c, q, [160, 33], out, lse, scale=4e-39)


@pytest.mark.gpu
@pytest.mark.parametrize("cache_type,q_type", [("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_attend_weights_of_rows_without_a_finite_score(cuda, cache_type, q_type, dim):
    """A head all of whose scores are minus infinity adds nothing to its kv head's weights: the
    other heads' shares arrive alone, and where every head is such a row the weights stay."""
    rng = np.random.default_rng(dim)
    lens = [150, 1, 31, 0]
    c = make_cache(rng, 4, 10, 16, 1, dim, DTYPES[cache_type])
    poison(c, lens, float("nan"))
    for b in (0, 2):  # positive against the one head's minus infinity
        page, place = row_index(c, b, torch.arange(lens[b]))
        c.k[page, :, place, 0] = c.k[page, :, place, 0].abs() + 0.125
    page, place = row_index(c, 1, [0])
    c.k[page, :, place] = 0
    c.k[page, :, place, 0] = float("inf")
    q = queries(rng, 4, 4, dim, DTYPES[q_type])
    q[:, 2] = 0
    q[:, 2, 0] = -float("inf")
    q[1] = 1
    q[1, :, 0] = -1
    plan = paged.AttentionPlan(c, 4, weights=True)
    before = torch.rand(4, 1, plan.max_len, device="cuda")
    weight = before.clone()
    out, lse = paged.attend(plan, q, int32(lens), return_lse=True, weight_in=weight, weight_out=weight)
    assert torch.count_nonzero(out[:, 2]) == 0 and (lse[:, 2] == -np.inf).all()
    assert torch.count_nonzero(out[1]) == 0 and (lse[1] == -np.inf).all()
    assert torch.equal(weight[1], before[1]) and torch.equal(weight[3], before[3])
    live = [0, 1, 3]
    lens[1] = 0  # nothing seen, as its output has it
    check(c, q[:, live], lens, out[:, live], lse[:, live], weight=weight, before=before)


@pytest.mark.gpu
@pytest.mark.parametrize("q_type", ["f32", "bf16"])
@pytest.mark.parametrize("dim,heads", [(64, 4), (64, 16), (128, 4), (256, 4)])
def test_attend_values_near_the_largest_bf16(cuda, q_type, dim, heads):
    """Values of up to about 2^116: their weighted sum is far from overflowing."""
    rng = np.random.default_rng(dim + heads)
    lens = [700, 0, 1, 33, 160]
    c = make_cache(rng, len(lens), 44, 16, 1, dim, torch.bfloat16)
    c.v.mul_(2.0 ** 114)
    poison(c, lens, float("nan"))
    q = queries(rng, len(lens), heads, dim, DTYPES[q_type])
    out, lse = paged.attend(paged.AttentionPlan(c, heads), q, int32(lens), return_lse=True)
    assert torch.isfinite(out).all()
    check(c, q, lens, out, lse)


@pytest.mark.gpu
@pytest.mark.parametrize("power", [125, -120])
@pytest.mark.parametrize("dim,heads", [(64, 4), (64, 16), (128, 4), (256, 4)])
def test_attend_keys_near_the_ends_of_bf16(cuda, dim, heads, power):
    """Keys near bf16's largest and near its smallest normal values, with queries that make
    ordinary scores of them."""
    rng = np.random.default_rng(dim + heads + power % 1000)
    lens = [700, 0, 1, 33, 160]
    c = make_cache(rng, len(lens), 44, 16, 1, dim, torch.bfloat16)
    c.k.mul_(2.0 ** power)
    poison(c, lens, float("nan"))
    q = queries(rng, len(lens), heads, dim, torch.float32) * 2.0 ** -power
    out, lse = paged.attend(paged.AttentionPlan(c, heads), q, int32(lens), return_lse=True)
    assert torch.isfinite(out).all()
    check(c, q, lens, out, lse)


@pytest.mark.gpu
def test_attend_front_end_refuses(cuda):
    rng = np.random.default_rng(16)
    c = make_cache(rng, 2, 2, 16, 2, 64, torch.float16)
    q, plan, lens = queries(rng, 2, 4, 64, torch.float16), paged.AttentionPlan(c, 4), int32([3, 4])
    w = torch.zeros(2, 2, 32, device="cuda")
    for bad in (dict(window=-1), dict(weight_in=w), dict(weight_out=w), dict(out=q[:1]), dict(lse=w)):
        with pytest.raises(ValueError):
            paged.attend(plan, q, lens, **bad)
    for bad_q in (q[:1], q.double(), q.cpu(), q.transpose(0, 1), q.repeat(1, 1, 2)[..., ::2]):
        with pytest.raises(ValueError):
            paged.attend(plan, bad_q, lens)
    for bad_lens in (lens.long(), lens.cpu(), lens[:1], int32([1, 2, 3, 4])[::2]):
        with pytest.raises(ValueError):
            paged.attend(plan, q, bad_lens)
    with pytest.raises(qgemv_b200.CudaError):
        paged.AttentionPlan(c, 3)
    assert paged.attend(plan, q, lens).shape == (2, 4, 64) and ops.get_error() == 0


@pytest.mark.gpu
def test_attend_strides_streams_and_lengths_past_the_table(cuda):
    rng = np.random.default_rng(6)
    c = make_cache(rng, 3, 4, 16, 2, 64, torch.float16, pad=8)
    wide = queries(rng, 3, 10, 64, torch.float16)
    q, out = wide[:, 2:6], torch.full((3, 12, 64), 5.0, dtype=torch.float16, device="cuda")
    plan = paged.AttentionPlan(c, 4)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    lens = int32([64, 1, 33])
    s.wait_stream(torch.cuda.current_stream())
    paged.attend(plan, q, lens, out=out[:, 4:8], stream=s)
    s.synchronize()
    check(c, q, [64, 1, 33], out[:, 4:8])
    assert (out[:, :4] == 5).all() and (out[:, 8:] == 5).all()
    ref = paged.attend(plan, q, int32([64, 0, 33]))
    got = paged.attend(plan, q, int32([65, -3, 33]))  # one past the table: cut; negative: none
    assert torch.equal(got, ref) and ops.get_error() == paged.QG_ERR_PAGE
    short = paged.AttentionPlan(c, 4, max_len=40)
    got = paged.attend(short, q, int32([64, 1, 33]))
    check(c, q, [40, 1, 33], got)
    assert ops.get_error() == paged.QG_ERR_PAGE


@pytest.mark.gpu
def test_attend_page_ids_outside_the_pool(cuda):
    """They are reported and never followed; other sequences are not touched by them, and ids
    past the length are not looked at."""
    rng = np.random.default_rng(7)
    c = make_cache(rng, 3, 4, 16, 2, 64, torch.float16)
    q, plan, lens = queries(rng, 3, 4, 64, torch.float16), paged.AttentionPlan(c, 4), int32([64, 20, 50])
    ref = paged.attend(plan, q, lens)
    c.table[1, 2:] = torch.tensor([-1, 2 ** 31 - 1], dtype=torch.int32)
    assert torch.equal(paged.attend(plan, q, lens), ref) and ops.get_error() == 0
    for bad in (-1, c.num_pages):
        c.table[0, 1] = bad
        got = paged.attend(plan, q, lens)
        assert torch.equal(got[1:], ref[1:]) and torch.isfinite(got).all()
        assert ops.get_error() == paged.QG_ERR_PAGE


@pytest.mark.gpu
def test_attend_offsets_past_32_bits(cuda):
    page, heads, dim = 64, 8, 128
    n = 2 ** 32 // (page * heads * dim * 2) + 3
    pool = torch.zeros(n, heads, page, dim, dtype=torch.float16, device="cuda")
    other = torch.zeros_like(pool)
    rng = np.random.default_rng(8)
    c = paged.PagedCache(pool, other, int32([[n - 1, n - 2]]))
    for p in (pool, other):
        p[-2:].normal_()
    q = queries(rng, 1, 16, dim, torch.float16)
    out = paged.attend(paged.AttentionPlan(c, 16), q, int32([128]))
    check(c, q, [128], out)


@pytest.mark.gpu
def test_attend_in_a_graph_follows_the_lengths(cuda):
    """One captured call serves growing sequences: lengths are read on the device."""
    rng = np.random.default_rng(9)
    c = make_cache(rng, 2, 40, 16, 2, 128, torch.float16)
    q, plan = queries(rng, 2, 16, 128, torch.float32), paged.AttentionPlan(c, 16)
    lens, out = int32([1, 0]), torch.empty(2, 16, 128, device="cuda")
    paged.attend(plan, q, lens, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        paged.attend(plan, q, lens, out=out)
    for n in ([1, 0], [300, 77], [640, 2], [0, 640]):
        lens.copy_(int32(n))
        graph.replay()
        check(c, q, n, out)


def _args():
    c = KvPagesC(64, 64, 1, 4, 16, 2, 64, 2048, 1024, 64, 64, 2, 2, 2)
    a = AttnC(64, 64, 1, 4, 256, 256, 64, 32, 0, 1.0, None, None, None, 0)
    return c, a


@pytest.mark.parametrize("what,field,value", [
    ("c", "k", None), ("c", "dtype", 0), ("c", "head_dim", 12), ("c", "slot_stride", 4), ("c", "page_size", 0),
    ("c", "table_pages", 2 ** 31 - 1), ("c", "head_stride", 1032), ("c", "slot_stride", 56), ("c", "page_stride", 1536),
    ("a", "q", None), ("a", "q", 8), ("a", "out", None), ("a", "out", 24), ("a", "dtype", -1), ("a", "dtype", 3),
    ("a", "n_q_heads", 0), ("a", "n_q_heads", 3), ("a", "q_stride", 4), ("a", "out_stride", 260), ("a", "lens", None),
    ("a", "max_len", 0), ("a", "max_len", 2 ** 31), ("a", "weight_in", 64), ("a", "weight_out", 64),
])
def test_attend_refuses_bad_arguments(what, field, value):
    c, a = _args()
    setattr(c if what == "c" else a, field, value)
    assert qgemv_b200.call("qg_paged_attn", ctypes.byref(c), ctypes.byref(a), 256, None) == INVALID_VALUE


def test_attend_refuses_bad_workspaces():
    c, a = _args()
    n = ctypes.c_size_t(0)
    for ws in (None, 128):
        assert qgemv_b200.call("qg_paged_attn", ctypes.byref(c), ctypes.byref(a), ws, None) == INVALID_VALUE
    size = ("qg_paged_attn_workspace_bytes", ctypes.byref(c))
    assert qgemv_b200.call(*size, 4, 32, 0, ctypes.byref(n)) == 0 and n.value >= 4096
    plain = n.value
    assert qgemv_b200.call(*size, 4, 32, 1, ctypes.byref(n)) == 0
    assert n.value >= plain + 2 * 4 * 32 * 4
    assert qgemv_b200.call(*size, 3, 32, 0, ctypes.byref(n)) == INVALID_VALUE
    assert qgemv_b200.call(*size, 4, 0, 0, ctypes.byref(n)) == INVALID_VALUE
    assert qgemv_b200.call(*size, 4, 32, 0, None) == INVALID_VALUE
