"""qg_qk_norm_rope_append (paged.qk_norm_rope_append) against the formula in 64 bits.

Tolerance of one rotated value y = a cos - b sin of normalised a, b: the fp32 work before the
rounding is a sum of up to 32 sequential and tree-added squares, a reciprocal root, two
products, and a fused rotation, together below 2^-20 of |a| + |b|; the rounding to the output
type is at most its unit roundoff of |y| (half a subnormal step below that).  Values that are
neither normalised nor rotated are rounded alone and have to be equal to the bit."""

import ctypes

import numpy as np
import pytest
import torch

import qgemv_b200
from paged_util import AppendC, DTYPES, INVALID_VALUE, KvPagesC, make_cache, row_index, TINY, UNIT
from qgemv_b200 import ops, paged


def formula(x, w, eps, rope, pos, pairs):
    """x [tokens, heads, dim] in float64 -> (y, |a| + |b|)."""
    if w is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
    y, size = x.copy(), np.abs(x)
    if rope is not None:
        rot = rope.shape[1]
        cos, sin = rope[pos][:, None, : rot // 2], rope[pos][:, None, rot // 2:]
        i = np.arange(rot // 2)
        a, b = (2 * i, 2 * i + 1) if pairs == "adjacent" else (i, i + rot // 2)
        y[..., a] = x[..., a] * cos - x[..., b] * sin
        y[..., b] = x[..., a] * sin + x[..., b] * cos
        size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    return y, size


def assert_near(got, want, size, dtype):
    got = got.double().cpu().numpy()
    tol = 2.0 ** -20 * size + UNIT[dtype] * np.abs(want) * (1 + 2.0 ** -19) + TINY[dtype]
    worst = np.max(np.abs(got - want) - tol) if got.size else -1.0
    assert worst <= 0, worst


def new_rows(rng, tokens, q_heads, kv_heads, dim, dtype, scale=3.0):
    """q, k, v as views of one fused projection."""
    qkv = torch.from_numpy(rng.standard_normal((tokens, (q_heads + 2 * kv_heads) * dim)) * scale).to(dtype).cuda()
    cut = q_heads * dim, (q_heads + kv_heads) * dim
    return (qkv[:, : cut[0]].unflatten(1, (q_heads, dim)), qkv[:, cut[0]: cut[1]].unflatten(1, (kv_heads, dim)),
            qkv[:, cut[1]:].unflatten(1, (kv_heads, dim)))


def f64(t):
    return t.double().cpu().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("tokens,q_heads,kv_heads,dim,rot,src,cache,page,order,pairs,norm", [
    (1, 64, 8, 128, 128, "f32", "f16", 16, "hsd", "adjacent", True),
    (1, 1, 1, 8, 0, "f16", "f16", 1, "hsd", "adjacent", True),       # the smallest head, no rotation
    (7, 5, 1, 64, 16, "f16", "f16", 5, "shd", "halves", True),       # one 8-value piece a half
    (33, 28, 4, 128, 128, "bf16", "bf16", 24, "shd", "halves", True),
    (3, 3, 3, 80, 32, "bf16", "f16", 16, "hsd", "adjacent", True),   # lanes without values
    (130, 6, 2, 112, 112, "f32", "bf16", 100, "shd", "halves", False),
    (9, 4, 2, 256, 64, "f16", "bf16", 32, "hsd", "halves", True),
    (9, 40, 8, 256, 256, "f32", "f16", 64, "shd", "adjacent", True),
    (517, 16, 1, 104, 48, "bf16", "bf16", 7, "hsd", "halves", True),
])
def test_append_matches_formula(cuda, tokens, q_heads, kv_heads, dim, rot, src, cache, page, order, pairs, norm):
    rng = np.random.default_rng(tokens * 31 + dim + rot)
    batch, capacity = 3, tokens + 40
    c = make_cache(rng, batch, -(-capacity // page), page, kv_heads, dim, DTYPES[cache], order)
    q, k, v = new_rows(rng, tokens, q_heads, kv_heads, dim, DTYPES[src])
    rope = paged.rope_table(4 * capacity, rot) if rot else None
    positions = rng.integers(0, 4 * capacity, tokens)
    seqs = rng.integers(0, batch, tokens)
    slots = np.zeros(tokens, dtype=np.int64)
    for b in range(batch):
        slots[seqs == b] = rng.permutation(capacity)[: np.sum(seqs == b)]
    if tokens > 2:
        positions[rng.integers(tokens)] = -1  # padding
        slots[rng.integers(tokens)] = -5      # nothing to append
    w = [torch.from_numpy(1 + 0.3 * rng.standard_normal(dim)).float().cuda() if norm else None for _ in range(2)]
    eps = 1e-5
    before = {n: getattr(c, n).clone() for n in "kv"}
    dev = [torch.from_numpy(a.astype(np.int32)).cuda() for a in (positions, slots, seqs)]
    out = paged.qk_norm_rope_append(c, q, k, v, rope, dev[0], slots=dev[1], seqs=dev[2], q_norm=w[0],
                                    k_norm=w[1], eps=eps, pairs=pairs)
    assert ops.get_error() == 0
    live, wn = positions >= 0, [None if x is None else f64(x) for x in w]
    r = None if rope is None else f64(rope)
    want, size = formula(f64(q)[live], wn[0], eps, r, positions[live], pairs)
    assert torch.count_nonzero(out[torch.from_numpy(~live).cuda()]) == 0
    assert_near(out[torch.from_numpy(live).cuda()], want, size, DTYPES[src])
    put = live & (slots >= 0)
    want, size = formula(f64(k)[put], wn[1], eps, r, positions[put], pairs)
    at = [row_index(c, int(b), [int(s)]) for b, s in zip(seqs[put], slots[put])]
    page_ids, places = torch.cat([a[0] for a in at]), torch.cat([a[1] for a in at])
    assert_near(c.k[page_ids, :, places], want, size, DTYPES[cache])
    assert torch.equal(c.v[page_ids, :, places], v[torch.from_numpy(put).cuda()].float().to(DTYPES[cache]))
    for n in "kv":  # every other row as it was
        keep = getattr(c, n).clone()
        keep[page_ids, :, places] = before[n][page_ids, :, places]
        assert torch.equal(keep, before[n])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_append_decode_defaults_in_place_on_a_stream(cuda, dtype):
    """No slots or seqs: token t is sequence t's next one, at its position.  q_out may be q;
    without norm and rotation q comes back to the bit."""
    rng = np.random.default_rng(5)
    c = make_cache(rng, 4, 3, 16, 2, 64, torch.float16)
    q, k, v = new_rows(rng, 4, 6, 2, 64, DTYPES[dtype])
    pos = torch.tensor([0, 17, 47, 31], dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    old = q.clone()
    out = paged.qk_norm_rope_append(c, q, k, v, None, pos, q_out=q, stream=s)
    s.synchronize()
    assert out is q and torch.equal(q, old)
    for b, p in enumerate(pos.tolist()):
        page, place = row_index(c, b, [p])
        assert torch.equal(c.k[page, :, place][0], k[b].to(torch.float16))
        assert torch.equal(c.v[page, :, place][0], v[b].to(torch.float16))
    rope, w = paged.rope_table(64, 64), torch.full((64,), 2.0, device="cuda")
    ref = paged.qk_norm_rope_append(c, q, k, v, rope, pos, q_norm=w)
    paged.qk_norm_rope_append(c, q, k, v, rope, pos, q_norm=w, q_out=q)
    assert torch.equal(ref, q)
    assert ops.get_error() == 0


@pytest.mark.gpu
def test_append_zero_rows_infinities_and_large_values(cuda):
    """A zero row stays zero (eps > 0); an infinity makes its own row NaN and no other; values
    whose squares would overflow fp16 normalise in fp32; values past the cache's type become
    its infinity."""
    rng = np.random.default_rng(6)
    c = make_cache(rng, 3, 1, 16, 2, 128, torch.float16)
    q, k, v = new_rows(rng, 3, 4, 2, 128, torch.float32)
    q[0] = 0
    q[1, 2, 7] = float("inf")
    k[2] *= 1e6
    v[2, 0, 3] = 1e6
    w, rope = torch.ones(128, device="cuda"), paged.rope_table(16, 128)
    pos = torch.tensor([0, 5, 9], dtype=torch.int32, device="cuda")
    out = paged.qk_norm_rope_append(c, q, k, v, rope, pos, q_norm=w, k_norm=w)
    assert torch.count_nonzero(out[0]) == 0
    assert not torch.isfinite(out[1, 2]).all() and torch.isfinite(out[1, [0, 1, 3]]).all()
    want, size = formula(f64(k)[2:], np.ones(128), 1e-5, f64(rope), np.array([9]), "adjacent")
    page, place = row_index(c, 2, [9])
    assert_near(c.k[page, :, place], want, size, torch.float16)
    assert torch.isinf(c.v[page, 0, place, 3]) and ops.get_error() == 0


@pytest.mark.gpu
def test_append_data_outside_the_cache_is_dropped(cuda):
    rng = np.random.default_rng(7)
    c = make_cache(rng, 2, 2, 16, 2, 64, torch.bfloat16)
    q, k, v = new_rows(rng, 1, 4, 2, 64, torch.bfloat16)
    rope = paged.rope_table(40, 64)
    before = {n: getattr(c, n).clone() for n in "kv"}

    def run(pos, slot, seq):
        ints = [torch.tensor([a], dtype=torch.int32, device="cuda") for a in (pos, slot, seq)]
        return paged.qk_norm_rope_append(c, q, k, v, rope, ints[0], slots=ints[1], seqs=ints[2]), ops.get_error()

    for pos, slot, seq, error in [(3, 32, 0, paged.QG_ERR_PAGE), (3, 2 ** 31 - 1, 0, paged.QG_ERR_PAGE),
                                  (3, 1, 2, paged.QG_ERR_PAGE), (3, 1, -1, paged.QG_ERR_PAGE),
                                  (40, 1, 0, paged.QG_ERR_POSITION)]:
        out, bits = run(pos, slot, seq)
        assert bits == error
        assert (torch.count_nonzero(out) == 0) == (error == paged.QG_ERR_POSITION)
    for bad in (-1, c.num_pages, 2 ** 31 - 1):
        c.table[1, 1] = bad
        assert run(3, 17, 1)[1] == paged.QG_ERR_PAGE
    assert run(3, 15, 1)[1] == 0  # its other page is sound
    page, place = row_index(c, 1, [15])
    assert torch.equal(c.v[page, :, place][0], v[0])
    before["v"][page, :, place], before["k"][page, :, place] = c.v[page, :, place], c.k[page, :, place]
    assert torch.equal(c.k, before["k"]) and torch.equal(c.v, before["v"])


@pytest.mark.gpu
def test_append_front_end_refuses(cuda):
    rng = np.random.default_rng(9)
    c = make_cache(rng, 2, 2, 16, 2, 64, torch.float16)
    q, k, v = new_rows(rng, 2, 4, 2, 64, torch.float16)
    pos, rope = torch.zeros(2, dtype=torch.int32, device="cuda"), paged.rope_table(8, 64)
    good = dict(q=q, k=k, v=v, rope=rope, positions=pos)
    before = c.k.clone()
    for bad in (dict(q=q.double()), dict(q=q.view(2, -1)), dict(k=k.float()), dict(k=k[:1]), dict(v=v.cpu()),
                dict(v=v.repeat(1, 1, 2)[..., ::2]), dict(positions=pos.long()), dict(positions=pos[:1]),
                dict(slots=pos.cpu()), dict(seqs=pos.repeat(2)[::2]), dict(rope=rope.half()), dict(pairs="both"),
                dict(q_norm=rope[0].half()), dict(k_norm=rope[0, :32]), dict(q_out=q.float())):
        with pytest.raises(ValueError):
            paged.qk_norm_rope_append(c, **(good | bad))
    for bad in (dict(rope=paged.rope_table(8, 24)), dict(rope=paged.rope_table(8, 80))):
        with pytest.raises(qgemv_b200.CudaError):
            paged.qk_norm_rope_append(c, **(good | bad))
    assert torch.equal(c.k, before) and ops.get_error() == 0


@pytest.mark.gpu
def test_append_offsets_past_32_bits(cuda):
    """Pools of more than 2^32 bytes: the last page's rows lie past any 32-bit offset."""
    page, heads, dim = 64, 8, 128
    n = 2 ** 32 // (page * heads * dim * 2) + 3
    pool = torch.zeros(n, heads, page, dim, dtype=torch.float16, device="cuda")
    other = torch.zeros_like(pool)
    table = torch.tensor([[n - 1, 0]], dtype=torch.int32, device="cuda")
    c = paged.PagedCache(pool, other, table)
    rng = np.random.default_rng(8)
    q, k, v = new_rows(rng, 1, 8, heads, dim, torch.float16)
    paged.qk_norm_rope_append(c, q, k, v, None, torch.tensor([63], dtype=torch.int32, device="cuda"))
    assert torch.equal(pool[n - 1, :, 63], k[0]) and torch.equal(other[n - 1, :, 63], v[0])
    assert torch.count_nonzero(pool[0]) == 0 and ops.get_error() == 0


def _args():
    c = KvPagesC(64, 64, 1, 4, 16, 2, 64, 2048, 1024, 64, 64, 2, 2, 2)
    a = AppendC(64, 64, 64, 64, 1, 2, 4, 256, 128, 128, 256, None, None, 1e-5, 64, 8, 64, 0, 64, None, None)
    return c, a


@pytest.mark.parametrize("what,field,value", [
    ("c", "k", None), ("c", "k", 72), ("c", "v", None), ("c", "table", None), ("c", "dtype", 0), ("c", "dtype", 3),
    ("c", "num_pages", 0), ("c", "page_size", 0), ("c", "n_kv_heads", 0), ("c", "head_dim", 0),
    ("c", "head_dim", 60), ("c", "head_dim", 264), ("c", "page_stride", 2044), ("c", "head_stride", 1020),
    ("c", "slot_stride", 68), ("c", "batch", 0), ("c", "table_pages", 0), ("c", "table_stride", 1),
    ("c", "batch", 1),  # two tokens, no seqs
    ("a", "q", None), ("a", "q", 72), ("a", "q_out", None), ("a", "q_out", 72), ("a", "k", None), ("a", "v", 72),
    ("a", "dtype", 3), ("a", "q_stride", 252), ("a", "v_stride", 124), ("a", "positions", None),
    ("a", "rope", None), ("a", "rope", 72), ("a", "rope_rows", 0), ("a", "rot_dim", 8), ("a", "rot_dim", 80),
    ("a", "pairs", 2), ("a", "q_norm", 72), ("a", "k_norm", 72), ("a", "n_q_heads", 65532),
])
def test_append_refuses_bad_arguments(what, field, value):
    """Returned before any launch (and any CUDA call)."""
    c, a = _args()
    setattr(c if what == "c" else a, field, value)
    assert qgemv_b200.call("qg_qk_norm_rope_append", ctypes.byref(c), ctypes.byref(a), None) == INVALID_VALUE


def test_append_without_tokens_or_structures():
    c, a = _args()
    assert qgemv_b200.call("qg_qk_norm_rope_append", None, ctypes.byref(a), None) == INVALID_VALUE
    assert qgemv_b200.call("qg_qk_norm_rope_append", ctypes.byref(c), None, None) == INVALID_VALUE
    a.tokens = 0
    assert qgemv_b200.call("qg_qk_norm_rope_append", ctypes.byref(c), ctypes.byref(a), None) == 0


def test_cache_front_end_refuses_what_is_not_on_a_device():
    pool, table = torch.zeros(2, 1, 16, 64, dtype=torch.float16), torch.zeros(1, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged.PagedCache(pool, pool, table)
    with pytest.raises(ValueError, match="one type and layout"):
        paged.PagedCache(pool, pool.float(), table)
