"""qg_qk_norm_rope_append8 (paged8.qk_norm_rope_append) against the formula in 64 bits.

Queries and, before they are quantised, keys: the 16-bit append's tolerance (2^-20 of the sizes that
a value is made of, and the rounding of the output type).  Values that are neither normalised nor
rotated are exact in fp32, so their scales and codes have to be equal.  A quantised key c s of x is
within half an e4m3 step of x, the step taken at |x| and that tolerance together, and its scale
the one of a largest value that is off by no more.  Codes that were there are rounded by a formula
without error: equal."""

import ctypes

import numpy as np
import pytest
import torch

import qgemv_b200
from paged8_util import (Append8C, BAD_PAGES, codes, e4m3, int32, make_cache, offsets, pages_c, places, values)
from paged_util import DTYPES, INVALID_VALUE, TINY, UNIT
from qgemv_b200 import ops, paged, paged8
from test_paged_append import formula, new_rows

f64 = lambda t: t.double().cpu().numpy()  # noqa: E731


def power_for(top):
    """The least power of two, within the scales' range, whose 448-fold reaches `top`."""
    if top <= 0:
        return 2.0 ** -60
    part, e = np.frexp(top)
    return 2.0 ** np.clip(e - 9 if part <= 0.875 else e - 8, -60, 60)


def step_at(size):
    return np.exp2(np.floor(np.log2(np.clip(size, 2.0 ** -6, 448.0))) - 3)


def check_pool(cache, name, before, x, size, lens, counts, err):
    """`before`: the codes and scales before the call; x [rows, heads, dim] new values, `size` what their
    errors are relative to, `err` how much."""
    page_size, block = cache.page_size, cache.block
    old_codes, old_scale = before
    got_codes, got_scale = f64(values(getattr(cache, name))), f64(getattr(cache, name + "_scale"))
    want_codes, want_scale = old_codes.copy(), old_scale.copy()
    mine = np.zeros(want_codes.shape[:3], dtype=bool)  # rows checked here
    row = 0
    for b, (n, new) in enumerate(zip(lens, counts)):
        slot = n - new
        while n > 0 and slot < n:
            page, place = int(cache.table[b, slot // page_size]), slot % page_size
            fill = min(block - place % block, n - slot)
            i, base = place // block, place // block * block
            for h in range(x.shape[1]):
                y, tol = x[row: row + fill, h], err * size[row: row + fill, h]
                top = np.abs(np.where(np.isfinite(y), y, 0)).max()
                slack = np.where(np.isfinite(tol), tol, 0).max()
                began = old_scale[page, h, i] if place % block else 0.0
                s = got_scale[page, h, i]
                assert max(power_for(top - slack), began) <= s <= max(power_for(top + slack), began), (name, b, h)
                want_scale[page, h, i] = s
                if place % block:
                    held = old_codes[page, h, base: base + block]
                    want_codes[page, h, base: base + block] = e4m3(held * (began / s))
                c = got_codes[page, h, place: place + fill]
                if err == 0:
                    assert np.array_equal(c, e4m3(y / s), equal_nan=True)
                else:
                    assert np.array_equal(np.isnan(c), np.isnan(y))
                    fine = np.isfinite(y)
                    off = np.abs(c - np.clip(y / s, -448, 448))[fine]
                    assert (off <= (step_at((np.abs(y) + tol) / s) / 2 + tol / s)[fine]).all()
                mine[page, h, place: place + fill] = True
            slot, row = slot + fill, row + fill
        row += new if n <= 0 else 0
    assert np.array_equal(got_codes[~mine], want_codes[~mine], equal_nan=True)
    assert np.array_equal(got_scale, want_scale)


def run(cache, rng, lens, counts, q_heads, src, rot, pairs, norm, ragged=True, pad=0, edit=None, positions=None):
    """One append of counts[b] rows that end at lens[b], checked; returns its rows."""
    heads, dim = cache.n_kv_heads, cache.head_dim
    tokens = sum(counts) + pad
    q, k, v = new_rows(rng, tokens, q_heads, heads, dim, DTYPES[src])
    if edit is not None:
        edit(q, k, v)
    if positions is None:
        positions = [(n - c + i + 5 * b) % 997 if n > 0 else -1
                     for b, (n, c) in enumerate(zip(lens, counts)) for i in range(c)] + [3] * pad
    rope = paged.rope_table(1000, rot) if rot else None
    wq, wk = (1 + 0.1 * torch.from_numpy(rng.standard_normal((2, dim))).float().cuda()) if norm else (None, None)
    before = {n: (f64(values(getattr(cache, n))), f64(getattr(cache, n + "_scale"))) for n in ("k", "v")}
    q_out = torch.full((tokens, q_heads, dim), 7.0, dtype=q.dtype, device="cuda")
    got = paged8.qk_norm_rope_append(cache, q, k, v, rope, int32(positions), int32(lens),
                                     offsets=offsets(counts) if ragged else None, q_norm=wq, k_norm=wk, eps=1e-5,
                                     pairs=pairs, q_out=q_out)
    assert got.data_ptr() == q_out.data_ptr()
    pos = np.array(positions)
    out = pos < 0 if rope is None else (pos < 0) | (pos >= 1000)
    use = np.where(out, 0, pos)
    r = None if rope is None else f64(rope)
    want, size = formula(f64(q), None if wq is None else f64(wq), 1e-5, r, use, pairs)
    keys, key_size = formula(f64(k), None if wk is None else f64(wk), 1e-5, r, use, pairs)
    vals = f64(v)
    want[out] = keys[out] = vals[out] = 0.0
    live = tokens - pad
    tol = 2.0 ** -20 * size + UNIT[q.dtype] * np.abs(want) * (1 + 2.0 ** -19) + TINY[q.dtype]
    assert np.nanmax(np.abs(f64(got)[:live] - want[:live]) - tol[:live], initial=-1.0) <= 0
    if ragged:
        assert (got[live:] == 7).all()  # rows of no sequence
    check_pool(cache, "k", before["k"], keys[:live], key_size[:live], lens, counts, 2.0 ** -20 if rot or norm else 0.0)
    check_pool(cache, "v", before["v"], vals[:live], np.abs(vals[:live]), lens, counts, 0.0)
    return q, k, v


CASES = [
    # q heads, kv heads, dim, rot, source, page, block, order, pairs, norm
    (64, 8, 128, 128, "f32", 32, 32, "hsd", "adjacent", True),
    (5, 1, 16, 0, "f16", 16, 16, "hsd", "adjacent", False),     # the smallest head, exact keys
    (6, 3, 48, 16, "f16", 48, 16, "shd", "halves", True),
    (28, 4, 80, 32, "bf16", 64, 32, "shd", "halves", True),
    (3, 1, 112, 112, "f32", 128, 128, "hsd", "halves", True),
    (16, 16, 64, 64, "bf16", 96, 32, "hsd", "adjacent", False),
    (4, 2, 256, 128, "f32", 128, 128, "shd", "adjacent", True),  # the most rows kept aside
    (4, 2, 256, 256, "bf16", 64, 64, "hsd", "halves", True),
    (2, 2, 128, 0, "bf16", 128, 64, "hsd", "adjacent", False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("q_heads,kv_heads,dim,rot,src,page,block,order,pairs,norm", CASES)
def test_append_prompts_and_chunks(cuda, q_heads, kv_heads, dim, rot, src, page, block, order, pairs, norm):
    """Ragged chunks one after another: fresh blocks, blocks begun before, whole pages, none."""
    rng = np.random.default_rng(dim + page + rot)
    c = make_cache(rng, 4, 700 // page + 1, page, block, kv_heads, dim, order)
    lens = [0, 0, 0, 0]
    for counts, pad in (([1, 0, 3, 2 * block], 0), ([block, 1, 2, 7], 2), ([3, 0, block - 5, 1], 1), ([300, 17, 1, 130], 0)):
        lens = [n + new for n, new in zip(lens, counts)]
        run(c, rng, lens, counts, q_heads, src, rot, pairs, norm, pad=pad)
    assert ops.get_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("q_heads,kv_heads,dim,rot,src,page,block,order,pairs,norm", CASES)
def test_append_one_row_a_sequence(cuda, q_heads, kv_heads, dim, rot, src, page, block, order, pairs, norm):
    """Decode steps; a row of padding (length 0, position -1) among them."""
    rng = np.random.default_rng(dim + page + rot + 1)
    c = make_cache(rng, 5, 3, page, block, kv_heads, dim, order, pad=16)
    lens = [1, block - 1, 0, block + 1, 2 * page]
    for _ in range(4):
        run(c, rng, lens, [1] * 5, q_heads, src, rot, pairs, norm, ragged=False)
        lens = [n + 1 if n else 0 for n in lens]
    run(c, rng, lens[:3] + [0, 0], [1] * 3, q_heads, src, rot, pairs, norm, ragged=False)  # fewer rows than sequences
    assert ops.get_error() == 0


@pytest.mark.gpu
def test_append_token_by_token_holds_what_one_call_writes(cuda):
    """Values of growing size: the scale grows often; the codes differ by a subnormal step at most."""
    rng = np.random.default_rng(1)
    for src in ("f32", "bf16"):
        whole = make_cache(rng, 2, 3, 64, 64, 2, 128)
        step = paged8.PagedCache8(*(codes(t).clone().view(torch.float8_e4m3fn) for t in (whole.k, whole.v)),
                                  whole.k_scale.clone(), whole.v_scale.clone(), whole.table)
        n = 150
        q, k, v = new_rows(rng, 2 * n, 2, 2, 128, DTYPES[src])
        grow = torch.exp2(torch.linspace(-12, 6, n, device="cuda")).to(k.dtype)[None, :, None, None]
        k, v = ((t.unflatten(0, (2, n)) * grow).contiguous() for t in (k, v))
        q, pos = q.unflatten(0, (2, n)), int32(list(range(n)))
        paged8.qk_norm_rope_append(whole, q.flatten(0, 1).contiguous(), k.flatten(0, 1), v.flatten(0, 1), None,
                                   int32([1] * 2 * n), int32([n, n]), offsets=offsets([n, n]))
        for i in range(n):
            paged8.qk_norm_rope_append(step, q[:, i].contiguous(), k[:, i].contiguous(), v[:, i].contiguous(), None,
                                       pos[i: i + 1].expand(2).contiguous(), int32([i + 1, i + 1]))
        for b in range(2):
            page, place = places(whole, b, torch.arange(n))
            for name in ("k", "v"):
                one, many = getattr(whole, name + "_scale"), getattr(step, name + "_scale")
                assert torch.equal(one[page, :, place // 64], many[page, :, place // 64])
                a, z = (values(getattr(c, name))[page, :, place] for c in (whole, step))
                # every growth rounds subnormal codes once more: half a step each, and the first rounding's
                assert ((a - z).abs() <= 2.0 ** -9 + 2.0 ** -9).all() and torch.equal(a[a.abs() >= 2], z[a.abs() >= 2])
    assert ops.get_error() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("src", ["f32", "bf16", "f16"])
def test_append_special_values(cuda, src):
    """Infinities saturate and set no scale, NaN stays NaN, zeros take the least scale, the ends of the
    scales' range hold, largest values that are 448 times a power of two fit exactly."""
    rng = np.random.default_rng(2)
    c = make_cache(rng, 6, 2, 32, 32, 2, 64)
    lens = [20] * 6

    def edit(q, k, v):
        for t in (k, v):
            t[:20] = 0.0
            t[21, 0, 3], t[22, 1, 5], t[23, 0, 0] = float("inf"), float("-inf"), float("nan")
            t[40:60] *= 2.0 ** -14 if src == "f16" else 2.0 ** -75
            if src != "f16":
                t[60:80] *= 2.0 ** 75
            t[80:100] = t[80:100].clamp(-3.4, 3.4)
            t[80, :, 1] = 3.5  # 448 * 2^-7
            t[100, :, 1] = -torch.nextafter(torch.tensor(3.5).bfloat16(), torch.tensor(9.0).bfloat16()).to(t.dtype) * 4

    run(c, rng, lens, [20] * 6, 2, src, 0, "adjacent", False, edit=edit)
    assert ops.get_error() == 0
    lens = [23] * 6
    run(c, rng, lens, [3] * 6, 2, src, 0, "adjacent", False)  # on top of them


@pytest.mark.gpu
def test_append_positions_and_padding(cuda):
    """A row without a position in the table gives zeros; of padding it says nothing."""
    rng = np.random.default_rng(3)
    c = make_cache(rng, 3, 2, 32, 16, 2, 64)
    run(c, rng, [4, 0, 7], [2, 2, 3], 4, "f32", 32, "adjacent", True, positions=[1000, 5, 1 << 30, -1, 0, -7, 8])
    assert ops.get_error() == paged.QG_ERR_POSITION
    run(c, rng, [5, 0, 8], [1, 1, 1], 4, "f16", 32, "halves", True, positions=[4, -1, -1], ragged=False)
    assert ops.get_error() == 0


@pytest.mark.gpu
def test_append_what_does_not_fit_is_dropped(cuda):
    rng = np.random.default_rng(4)
    c = make_cache(rng, 3, 2, 32, 16, 1, 64)
    q, k, v = new_rows(rng, 9, 2, 1, 64, torch.float32)
    pos = int32([0] * 9)
    before = codes(c.k).clone(), codes(c.v).clone(), c.k_scale.clone(), c.v_scale.clone()

    def same():
        return all(torch.equal(x, y) for x, y in zip(before, (codes(c.k), codes(c.v), c.k_scale, c.v_scale)))

    for lens, counts in (([65, 0, 0], [9, 0, 0]), ([8, 0, 0], [9, 0, 0]), ([-5, -1, 0], [3, 3, 3]), ([5, 5, 5], [0, 0, 0])):
        paged8.qk_norm_rope_append(c, q, k, v, None, pos, int32(lens), offsets=offsets(counts))
        assert same() and ops.get_error() == (paged.QG_ERR_PAGE if max(lens) > 5 else 0)
    for bad in ([0, 12, 12, 12], [3, 1, 1, 1], [-1, 0, 0, 0], [0, 0, -4, 0]):
        paged8.qk_norm_rope_append(c, q, k, v, None, pos, int32([0, 0, 0]), offsets=int32(bad))
        assert same() and ops.get_error() == paged.QG_ERR_PAGE
    table = c.table.clone()
    c.table.fill_(c.num_pages)
    paged8.qk_norm_rope_append(c, q, k, v, None, pos, int32([30, 4, 0]), offsets=offsets([5, 4, 0]))
    assert same() and ops.get_error() == paged.QG_ERR_PAGE
    c.table.copy_(table)
    empty = q[:0]
    assert paged8.qk_norm_rope_append(c, empty, k[:0], v[:0], None, pos[:0], int32([0, 0, 0])).shape == (0, 2, 64)
    assert same() and ops.get_error() == 0


@pytest.mark.gpu
def test_append_many_sequences_long_tables_and_offsets_past_32_bits(cuda):
    rng = np.random.default_rng(5)
    counts = [int(n) for n in rng.integers(0, 3, 300)]
    lens = [n + int(rng.integers(0, 60)) if n else 0 for n in counts]
    c = make_cache(rng, 300, 2, 32, 16, 1, 64)
    run(c, rng, lens, counts, 3, "f16", 64, "adjacent", True)
    heads, page, dim = 8, 128, 128
    n = 2 ** 32 // (heads * page * dim) + 3
    pool = torch.zeros(2, n, heads, page, dim, dtype=torch.uint8, device="cuda")
    scale = torch.zeros(2, n, heads, 1, device="cuda")
    c = paged8.PagedCache8(*(p.view(torch.float8_e4m3fn) for p in pool), *scale, int32([[n - 1, n - 2]]))
    q, k, v = new_rows(rng, 140, 8, heads, dim, torch.float16)
    paged8.qk_norm_rope_append(c, q, k, v, None, int32([0] * 140), int32([140]), offsets=offsets([140]))
    for t, name in ((k, "k"), (v, "v")):
        got = torch.cat([pool[int(name == "v"), n - 1], pool[int(name == "v"), n - 2, :, :12]], 1)
        s = scale[int(name == "v"), [n - 1, n - 2]]
        s = torch.cat([s[:1].expand(128, heads, 1), s[1:].expand(12, heads, 1)])
        want = (t.float() / s).to(torch.float8_e4m3fn)
        assert torch.equal(got.transpose(0, 1), codes(want))
    assert ops.get_error() == 0


@pytest.mark.gpu
def test_append_streams_and_graphs(cuda):
    """One captured call serves growing sequences; a call on another stream uses that stream."""
    rng = np.random.default_rng(6)
    c = make_cache(rng, 2, 2, 64, 32, 2, 128)
    same = paged8.PagedCache8(*(codes(t).clone().view(torch.float8_e4m3fn) for t in (c.k, c.v)), c.k_scale.clone(),
                              c.v_scale.clone(), c.table)
    q, k, v = new_rows(rng, 2, 4, 2, 128, torch.float32)
    rope, pos, lens = paged.rope_table(200, 64), int32([0, 9]), int32([0, 9])
    out = torch.empty_like(q.contiguous())
    paged8.qk_norm_rope_append(c, q, k, v, rope, pos, int32([0, 0]), q_out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lens += 1
        pos += 1
        paged8.qk_norm_rope_append(c, q, k, v, rope, pos, lens, q_out=out)
    s = torch.cuda.Stream()
    for i in range(1, 70):
        graph.replay()
        s.wait_stream(torch.cuda.current_stream())
        ref = paged8.qk_norm_rope_append(same, q, k, v, rope, int32([i, 9 + i]), int32([i, 9 + i]), stream=s)
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(ref, out)
    torch.cuda.synchronize()
    assert torch.equal(codes(c.k), codes(same.k)) and torch.equal(codes(c.v), codes(same.v))
    assert torch.equal(c.k_scale, same.k_scale) and torch.equal(c.v_scale, same.v_scale) and ops.get_error() == 0


@pytest.mark.gpu
def test_append_front_end_refuses(cuda):
    rng = np.random.default_rng(7)
    c = make_cache(rng, 2, 2, 32, 16, 2, 64)
    q, k, v = (t.contiguous() for t in new_rows(rng, 2, 4, 2, 64, torch.float16))
    pos, lens = int32([0, 0]), int32([1, 1])
    ok = dict(q=q, k=k, v=v, rope=None, positions=pos, lens=lens)
    bad = [dict(q=q[0]), dict(q=q.double()), dict(q=q.cpu()), dict(k=k[:1]), dict(k=k.float()), dict(v=v[..., :32]),
           dict(v=v.transpose(0, 1)), dict(positions=pos.long()), dict(positions=pos[:1]), dict(lens=lens[:1]),
           dict(lens=lens.long()), dict(lens=lens.cpu()), dict(offsets=lens), dict(offsets=int32([0, 1, 2]).long()),
           dict(q_norm=torch.ones(32, device="cuda")), dict(rope=torch.ones(4, device="cuda")), dict(pairs="both"),
           dict(q_out=q[:1]), dict(q=q.repeat(2, 1, 1), k=k.repeat(2, 1, 1), v=v.repeat(2, 1, 1), positions=int32([0] * 4))]
    for b in bad:
        with pytest.raises(ValueError):
            paged8.qk_norm_rope_append(c, **(ok | b))
    with pytest.raises(qgemv_b200.CudaError):
        paged8.qk_norm_rope_append(c, **(ok | dict(rope=torch.ones(4, 24, device="cuda"))))
    assert paged8.qk_norm_rope_append(c, **ok).shape == q.shape and ops.get_error() == 0


@pytest.mark.gpu
def test_cache_refuses(cuda):
    pool = torch.zeros(4, 2, 32, 64, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    scale, table = torch.zeros(4, 2, 2, device="cuda"), int32([[0, 1]])
    assert paged8.PagedCache8(pool, pool, scale, scale, table).block == 16
    half = codes(pool).half()
    for args in ((half, half, scale, scale, table), (pool, pool[:3], scale, scale, table),
                 (pool, pool, scale[:3], scale[:3], table), (pool, pool, scale, scale.double(), table),
                 (pool, pool, scale[..., :0], scale[..., :0], table), (pool, pool, scale, scale, table.long()),
                 (pool, pool, scale, scale, table.cpu()), (pool, pool, scale.expand(4, 2, 2)[..., :1].expand(4, 2, 5),
                                                           scale[..., :1].expand(4, 2, 5), table)):
        with pytest.raises(ValueError):
            paged8.PagedCache8(*args)
    c = paged8.PagedCache8(pool, pool, scale, scale, table)
    with pytest.raises(AttributeError):
        c.k = pool
    with pytest.raises(ValueError):
        paged8.PagedCache8.empty(4, 2, 32, 64, 1, 2, block=24)
    odd = paged8.PagedCache8(pool, pool, scale[..., :1].contiguous(), scale[..., :1].contiguous(), table)
    assert odd.block == 32


def _args():
    return pages_c(), Append8C(64, 64, 64, 64, 0, 2, 4, 256, 128, 128, 256, None, None, 1e-5, None, 0, 0, 0, 64, 64, None)


@pytest.mark.parametrize("field,value", BAD_PAGES)
def test_append_refuses_bad_caches(field, value):
    c, a = _args()
    setattr(c, field, value)
    assert qgemv_b200.call("qg_qk_norm_rope_append8", ctypes.byref(c), ctypes.byref(a), None) == INVALID_VALUE


@pytest.mark.parametrize("field,value", [
    ("q", None), ("q", 8), ("k", None), ("k", 24), ("v", None), ("v", 8), ("q_out", None), ("q_out", 72), ("dtype", 3),
    ("dtype", -1), ("tokens", 2 ** 31), ("tokens", 3), ("n_q_heads", 65536), ("q_stride", 258), ("k_stride", 130),
    ("v_stride", 129), ("q_out_stride", 2), ("q_norm", 8), ("k_norm", 4), ("rot_dim", 16), ("rot_dim", 8), ("pairs", 2),
    ("positions", None), ("lens", None),
])
def test_append_refuses_bad_arguments(field, value):
    c, a = _args()
    setattr(a, field, value)
    assert qgemv_b200.call("qg_qk_norm_rope_append8", ctypes.byref(c), ctypes.byref(a), None) == INVALID_VALUE


def test_append_of_nothing_does_nothing():
    c, a = _args()
    a.tokens = 0
    assert qgemv_b200.call("qg_qk_norm_rope_append8", ctypes.byref(c), ctypes.byref(a), None) == 0
    assert qgemv_b200.call("qg_qk_norm_rope_append8", None, ctypes.byref(a), None) == INVALID_VALUE
    assert qgemv_b200.call("qg_qk_norm_rope_append8", ctypes.byref(c), None, None) == INVALID_VALUE


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dim,rot,block,src,pairs", [
    (9, 128, 128, 32, "f32", "halves"), (9, 128, 64, 16, "bf16", "adjacent"), (17, 48, 48, 64, "f16", "halves"),
    (5, 256, 256, 128, "f16", "adjacent"), (1, 16, 0, 16, "f32", "adjacent"),
])
def test_append_one_row_a_sequence_equals_the_ragged_call(cuda, heads, dim, rot, block, src, pairs):
    """Without offsets a row is a warp's, with them a block is a CTA's: the same bits, while scales grow, where
    sequences are padding or have a bad page, and where a position is none."""
    rng = np.random.default_rng(6)
    one = make_cache(rng, 7, 2, 128, block, heads, dim)
    one.table[3, 0] = one.num_pages
    ragged = paged8.PagedCache8(*(codes(t).clone().view(torch.float8_e4m3fn) for t in (one.k, one.v)),
                                one.k_scale.clone(), one.v_scale.clone(), one.table)
    rope = paged.rope_table(60, rot) if rot else None
    norm = 1 + 0.1 * torch.from_numpy(rng.standard_normal(dim)).float().cuda()
    for i in range(block - 3, block + 40):
        q, k, v = new_rows(rng, 7, heads + 2, heads, dim, DTYPES[src])
        k, v = k * 2.0 ** (i % 23 - 12), v * 2.0 ** (i % 19 - 12)
        lens, pos = int32([i, 1, 0, 5, i + 100, 3 * i, i]), int32([i % 60, 1, 2, 3, -1, 59, 60 if i % 2 else 0])
        got = [paged8.qk_norm_rope_append(c, q, k, v, rope, pos, lens, offsets=at, q_norm=norm, pairs=pairs)
               for c, at in ((one, None), (ragged, offsets([1] * 7)))]
        assert torch.equal(*got)
        for name in ("k", "v"):
            assert torch.equal(codes(getattr(one, name)), codes(getattr(ragged, name)))
            assert torch.equal(getattr(one, name + "_scale"), getattr(ragged, name + "_scale"))
        assert ops.get_error() == paged.QG_ERR_PAGE | (paged.QG_ERR_POSITION if rot and i % 2 else 0)


@pytest.mark.gpu
@pytest.mark.parametrize("block", [16, 64])
def test_append_reports_what_does_not_fit_behind_the_last_row(cuda, block):
    """Many sequences, rows of the first three alone: offsets and lengths of the others are looked at too."""
    rng = np.random.default_rng(8)
    batch = 400
    c = make_cache(rng, batch, 1, 64, block, 1, 64)
    q, k, v = new_rows(rng, 3, 2, 1, 64, torch.float16)
    pos = int32([0] * 3)
    off, lens = np.array([0, 1, 2] + [3] * (batch - 2)), np.array([1, 1, 1] + [0] * (batch - 3))
    paged8.qk_norm_rope_append(c, q, k, v, None, pos, int32(lens.tolist()), offsets=int32(off.tolist()))
    assert ops.get_error() == 0
    for at in (60, 127, 128, 129, 300, 399):
        bad = off.copy()
        bad[at] = 2
        paged8.qk_norm_rope_append(c, q, k, v, None, pos, int32(lens.tolist()), offsets=int32(bad.tolist()))
        assert ops.get_error() == paged.QG_ERR_PAGE, at
        long = lens.copy()
        long[at] = 65
        paged8.qk_norm_rope_append(c, q, k, v, None, pos, int32(long.tolist()), offsets=int32(off.tolist()))
        assert ops.get_error() == paged.QG_ERR_PAGE, at
