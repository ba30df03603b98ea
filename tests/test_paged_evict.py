"""qg_kv_evict (paged.evict): kept slots, moved rows, weights and lengths are all exact, so every
comparison is for equality with a stable sort."""

import ctypes

import numpy as np
import pytest
import torch

import qgemv_b200
from paged_util import DTYPES, EvictC, INVALID_VALUE, KvPagesC, make_cache, row_index
from qgemv_b200 import ops, paged


def int32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def choice(w, n, budget, sink, recent):
    """Kept slots of one head: numpy, ties to the lower slot, NaN last."""
    if n <= budget:
        return np.arange(n)
    middle = np.arange(sink, n - recent)
    rank = np.where(np.isnan(w[middle]), -np.inf, w[middle])
    order = np.lexsort((middle, np.isnan(w[middle]), -rank))  # weight, NaN after -inf, then slot
    best = middle[order[: budget - sink - recent]]
    return np.sort(np.concatenate([np.arange(sink), best, np.arange(n - recent, n)]))


def check(cache, old, table, kept, weight_old, weight_new, lens_old, lens_new, budget, sink, recent):
    """`old`: the pools before; `table`: the pages that hold the rows afterwards."""
    w_old, w_new = weight_old.cpu().numpy(), weight_new.cpu().numpy()
    kept = kept.cpu().numpy()
    after = paged.PagedCache(cache.k, cache.v, table)
    for b, n in enumerate(lens_old):
        m = min(n, budget)
        assert lens_new[b].item() == m
        for h in range(cache.n_kv_heads):
            want = choice(w_old[b, h], n, budget, sink, recent)
            assert np.array_equal(kept[b, h, :m], want) and (kept[b, h, m:] == -1).all()
            assert np.array_equal(w_new[b, h, :m], w_old[b, h][want], equal_nan=True)
            assert (w_new[b, h, m:] == 0).all()
            (sp, ss), (dp, ds) = row_index(cache, b, want), row_index(after, b, np.arange(m))
            for name, pool in (("k", cache.k), ("v", cache.v)):
                assert torch.equal(pool[dp, h, ds], old[name][sp, h, ss])


def weights(rng, shape, lens):
    """Heavy-tailed sums with many ties: zeros and repeated values."""
    w = np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
    w[rng.random(shape) < 0.3] = 0.0
    w[rng.random(shape) < 0.2] = 0.5
    for b, n in enumerate(lens):
        w[b, :, n:] = 0
    return torch.from_numpy(w).cuda()


CASES = [
    # lengths, budget, sink, recent, kv heads, dim, page, order
    ([1, 0, 3, 2], 2, 0, 1, 1, 8, 1, "hsd"),
    ([100, 99, 64, 65, 0], 64, 4, 16, 2, 64, 16, "hsd"),
    ([700, 513, 514], 513, 0, 0, 3, 80, 24, "shd"),        # the budget ends inside a page
    ([1500], 600, 300, 300, 2, 128, 7, "shd"),             # nothing to choose
    ([1500, 40], 1, 0, 0, 2, 112, 100, "hsd"),
    ([1500, 1499], 1499, 1, 1, 1, 256, 64, "hsd"),         # one goes
    ([9000, 5000, 2049], 2048, 4, 511, 2, 64, 32, "shd"),  # several chunks of rows
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lens,budget,sink,recent,heads,dim,page,order", CASES)
def test_evict_keeps_the_heaviest(cuda, lens, budget, sink, recent, heads, dim, page, order, in_place, dtype):
    rng = np.random.default_rng(budget + dim)
    pages, to = -(-max(lens) // page) + 1, -(-min(budget, max(lens)) // page)
    both = make_cache(rng, len(lens), pages + to, page, heads, dim, DTYPES[dtype], order)
    c = paged.PagedCache(both.k, both.v, both.table[:, :pages])
    table = both.table[:, pages:]
    old = {"k": c.k.clone(), "v": c.v.clone()}
    width = max(lens) + 3
    w = weights(rng, (len(lens), heads, width), lens)
    w0, ln = w.clone(), int32(lens)
    if in_place:
        kept, new = paged.evict(c, ln, w, budget, sink=sink, recent=recent)
        assert new is ln
        check(c, old, c.table, kept, w0, w, lens, new, budget, sink, recent)
    else:
        w1 = torch.full_like(w, 3.0)
        kept, new = paged.evict(c, ln, w, budget, sink=sink, recent=recent, new_table=table, weight_out=w1)
        check(c, old, table, kept, w0, w1, lens, new, budget, sink, recent)
        assert torch.equal(w, w0) and ln.tolist() == lens
        for name in ("k", "v"):  # the old pages keep their rows
            page_ids = c.table.long().flatten()
            assert torch.equal(getattr(c, name)[page_ids], old[name][page_ids])
    assert ops.get_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
def test_evict_weights_apart_from_rows(cuda, in_place):
    """Rows in place with new weights elsewhere, and rows elsewhere with weights in place: the
    first kept slots do not move, their weights still have to."""
    rng = np.random.default_rng(3)
    lens, budget = [1500, 700, 90], 600
    c = make_cache(rng, 3, 94 if in_place else 134, 16, 2, 128, torch.float16)
    c, table = paged.PagedCache(c.k, c.v, c.table[:, :94]), c.table[:, :94] if in_place else c.table[:, 94:]
    old = {"k": c.k.clone(), "v": c.v.clone()}
    w = weights(rng, (3, 2, 1500), lens)
    w[:, :, :300] += 1e5  # the first slots stay where they are
    w0, ln, out = w.clone(), int32(lens), torch.full_like(w, 9.0) if in_place else w
    kept, new = paged.evict(c, ln, w, budget, recent=10, new_table=None if in_place else table, weight_out=out)
    check(c, old, table, kept, w0, out, lens, new, budget, 0, 10)
    assert not in_place or torch.equal(w, w0)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["zeros", "alike", "special", "narrow", "rising", "falling"])
@pytest.mark.parametrize("n", [1000, 60000])  # keys held in shared memory, and read again
def test_evict_ties_and_special_weights(cuda, kind, n):
    rng = np.random.default_rng(n)
    c = make_cache(rng, 1, n // 100 + 1, 100, 2, 8, torch.float16)
    w = np.zeros((1, 2, n), dtype=np.float32)
    if kind == "alike":
        w[:] = 0.25
    elif kind == "special":
        w[:] = rng.choice(np.array([np.nan, -np.inf, np.inf, -0.0, 0.0, -1.5, 1e-45, -1e-45, 3e38], np.float32), w.shape)
    elif kind == "narrow":  # they differ in the last bits alone
        w[:] = (0x3F800000 + rng.integers(0, 50, w.shape)).astype(np.uint32).view(np.float32)
    elif kind != "zeros":
        w[:] = np.arange(n) * (1 if kind == "rising" else -1)
    old, w = {"k": c.k.clone(), "v": c.v.clone()}, torch.from_numpy(w).cuda()
    for budget, sink, recent in ((n * 2 // 3, 3, 50), (n // 7, 0, 0)):
        w1, kv = w.clone(), {"k": c.k.clone(), "v": c.v.clone()}
        kept, new = paged.evict(c, int32([n]), w1, budget, sink=sink, recent=recent)
        check(c, old, c.table, kept, w, w1, [n], new, budget, sink, recent)
        c.k.copy_(kv["k"]), c.v.copy_(kv["v"])


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("lens,width,budget", [
    ([50000, 49999, 7, 0, 3000] * 8, 50000, 2500),  # a line a CTA: more lines than SMs, rows wider than it keeps
    ([400000], 400003, 100000),                     # a cluster of 8 with more than it keeps
])
def test_evict_keys_past_shared_memory(cuda, lens, width, budget, in_place):
    """Selections whose keys do not stay in shared memory read the weights again in every pass."""
    rng = np.random.default_rng(width)
    page, heads, dim = 100, 2, 8
    pages, to = -(-max(lens) // page), -(-budget // page)
    both = make_cache(rng, len(lens), pages + to, page, heads, dim, torch.float16)
    c, table = paged.PagedCache(both.k, both.v, both.table[:, :pages]), both.table[:, pages:]
    old = {"k": c.k.clone(), "v": c.v.clone()}
    w = weights(rng, (len(lens), heads, width), lens)
    w0, ln = w.clone(), int32(lens)
    if in_place:
        kept, new = paged.evict(c, ln, w, budget, sink=3, recent=201)
        check(c, old, c.table, kept, w0, w, lens, new, budget, 3, 201)
    else:
        w1 = torch.full_like(w, 3.0)
        kept, new = paged.evict(c, ln, w, budget, sink=3, recent=201, new_table=table, weight_out=w1)
        check(c, old, table, kept, w0, w1, lens, new, budget, 3, 201)
        assert torch.equal(w, w0) and ln.tolist() == lens
    assert ops.get_error() == 0


@pytest.mark.gpu
def test_evict_twice_and_on_a_stream(cuda):
    """A second call at the same budget changes nothing; eviction, growth and eviction again."""
    rng = np.random.default_rng(1)
    c = make_cache(rng, 2, 10, 32, 2, 64, torch.bfloat16)
    lens, budget = [300, 120], 100
    w, ln = weights(rng, (2, 2, c.capacity), lens), int32(lens)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    paged.evict(c, ln, w, budget, sink=2, recent=20, stream=s)
    s.synchronize()
    state = [t.clone() for t in (c.k, c.v, w, ln)]
    kept, _ = paged.evict(c, ln, w, budget, sink=2, recent=20)
    assert torch.equal(kept, torch.arange(100, device="cuda", dtype=torch.int32).expand(2, 2, 100))
    assert all(torch.equal(a, b) for a, b in zip(state, (c.k, c.v, w, ln)))
    ln += 7
    w[:, :, 100:107] = 1e6  # new slots that matter
    kept, _ = paged.evict(c, ln, w, budget, sink=0, recent=0)
    assert (kept[:, :, -7:] == torch.arange(100, 107, device="cuda")).all() and ops.get_error() == 0


@pytest.mark.gpu
def test_evict_data_outside_the_cache(cuda):
    """Lengths past the table are cut and reported; bad page ids are reported, rows written to
    them dropped, rows read from them zero."""
    rng = np.random.default_rng(2)
    c = make_cache(rng, 2, 4, 16, 1, 64, torch.float16)
    w = torch.rand(2, 1, 70, device="cuda")
    kept, new = paged.evict(c, int32([65, -1]), w.clone(), 70)
    assert new.tolist() == [64, 0] and ops.get_error() == paged.QG_ERR_PAGE
    c.table[0, 3] = c.num_pages
    before = c.k.clone()
    kept, new = paged.evict(c, int32([64, 64]), w.clone(), 20, recent=20)
    assert new.tolist() == [20, 20] and ops.get_error() == paged.QG_ERR_PAGE
    page, place = row_index(c, 0, torch.arange(20))
    assert torch.equal(kept[0, 0].cpu(), torch.arange(44, 64, dtype=torch.int32))
    src = before[row_index(c, 0, torch.arange(44, 48))[0], 0, row_index(c, 0, torch.arange(44, 48))[1]]
    assert torch.equal(c.k[page[:4], 0, place[:4]], src)
    assert torch.count_nonzero(c.k[page[4:], 0, place[4:]]) == 0


@pytest.mark.gpu
def test_evict_front_end_refuses(cuda):
    rng = np.random.default_rng(3)
    c = make_cache(rng, 2, 4, 16, 2, 64, torch.float16)
    lens, w, table = int32([20, 30]), torch.zeros(2, 2, 64, device="cuda"), int32([[0], [1]])
    for bad in (dict(new_table=table), dict(new_table=table.long(), weight_out=w), dict(new_table=table[:1], weight_out=w),
                dict(lens_out=lens.long()), dict(weight_out=w[:, :1]), dict(kept=int32([1]))):
        with pytest.raises(ValueError):
            paged.evict(c, lens, w, 10, **bad)
    for bad in (w[:, :, ::2], w.half(), w.cpu(), w[0]):
        with pytest.raises(ValueError):
            paged.evict(c, lens, bad, 10)
    for bad in (dict(sink=8, recent=8), dict(sink=-1), dict(recent=11)):
        with pytest.raises(qgemv_b200.CudaError):
            paged.evict(c, lens, w, 10, **bad)
    with pytest.raises(qgemv_b200.CudaError):  # 16 slots are not room for 17
        paged.evict(c, lens, w, 17, new_table=table, weight_out=w.clone())
    assert lens.tolist() == [20, 30] and ops.get_error() == 0


@pytest.mark.gpu
def test_evict_offsets_past_32_bits(cuda):
    page, heads, dim = 64, 8, 128
    n = 2 ** 32 // (page * heads * dim * 2) + 3
    pool = torch.zeros(n, heads, page, dim, dtype=torch.float16, device="cuda")
    other = torch.zeros_like(pool)
    c = paged.PagedCache(pool, other, int32([[0, n - 1]]))
    pool[n - 1].normal_(), other[n - 1].normal_()
    w = torch.zeros(1, heads, 128, device="cuda")
    w[:, :, 70:100] = 1
    paged.evict(c, int32([128]), w, 30)
    assert torch.equal(pool[0, :, :30], pool[n - 1, :, 6:36]) and torch.equal(other[0, :, :30], other[n - 1, :, 6:36])


def _args():
    c = KvPagesC(64, 64, 1, 4, 16, 2, 64, 2048, 1024, 64, 64, 2, 2, 2)
    return c, EvictC(64, 64, 64, 64, 32, 32, 16, 4, 4, 64, 64, 1, 1)


@pytest.mark.parametrize("what,field,value", [
    ("c", "v", None), ("c", "dtype", 0), ("c", "head_dim", 4), ("c", "batch", 65536),
    ("e", "lens", None), ("e", "lens_out", None), ("e", "weight", None), ("e", "weight_out", None), ("e", "kept", None),
    ("e", "max_len", 0), ("e", "max_len", 33), ("e", "weight_stride", 31), ("e", "budget", 0), ("e", "budget", 7),
    ("e", "sink", 13), ("e", "recent", 2 ** 32 - 1), ("e", "budget", 17), ("e", "new_table_stride", 0),
])
def test_evict_refuses_bad_arguments(what, field, value):
    c, e = _args()
    setattr(c if what == "c" else e, field, value)
    assert qgemv_b200.call("qg_kv_evict", ctypes.byref(c), ctypes.byref(e), None) == INVALID_VALUE
