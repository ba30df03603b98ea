"""The paged cache operators as a decode loop uses them (examples/paged_decode.py), step by
step against 64-bit arithmetic on the block's own projections: append, attention with summed
weights, eviction in place and decoding on in the reused slots."""

import sys

import numpy as np
import pytest
import torch

from conftest import REPO
from qgemv_b200 import ops, packs, paged

sys.path.insert(0, str(REPO / "examples"))


def turned(x, w, rope, pos):
    """Norm and rotation of [heads, dim] rows in float64 (neighbouring pairs)."""
    x = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-5) * w
    half = rope.shape[1] // 2
    cos, sin = rope[pos, :half], rope[pos, half:]
    y = np.empty_like(x)
    y[:, 0::2], y[:, 1::2] = x[:, 0::2] * cos - x[:, 1::2] * sin, x[:, 0::2] * sin + x[:, 1::2] * cos
    return y


@pytest.mark.gpu
@pytest.mark.parametrize("requests", [1, 3, 6])  # GEMV, multi-vector GEMV, tensor-core tiles
def test_decode_with_eviction_follows_64_bits(cuda, requests):
    from paged_decode import Block

    budget, slack, sink, recent = 24, 8, 2, 6
    block = Block(requests, hidden=512, q_heads=8, kv_heads=2, head_dim=64, budget=budget, slack=slack,
                  page_size=5, sink=sink, recent=recent, max_positions=256)
    f64 = lambda t: t.detach().double().cpu().numpy()  # noqa: E731
    rope, qw, kw = f64(block.rope), f64(block.q_norm), f64(block.k_norm)
    # what the cache should hold: keys, values and summed weights of every request and head
    rows = [[dict(k=[], v=[], w=[]) for _ in range(2)] for _ in range(requests)]
    gen = torch.Generator(device="cuda")
    gen.manual_seed(requests)
    evicted = 0
    for step in range(60):
        x = torch.randn(requests, 512, generator=gen, device="cuda")
        got = block.step(x)
        if got["kept"] is not None:
            evicted += 1
            kept = got["kept"].cpu().numpy()
            for b in range(requests):
                for h in range(2):
                    r, keep = rows[b][h], kept[b, h]
                    n, w = len(r["w"]), np.array(r["w"])
                    assert (np.diff(keep) > 0).all() and set(range(sink)) | set(range(n - recent, n)) <= set(keep)
                    gone = np.setdiff1d(np.arange(n), keep)
                    middle = keep[(keep >= sink) & (keep < n - recent)]
                    # every slot that stayed outweighs every slot that went, to the sums' precision
                    assert w[middle].min() >= w[gone].max() - 1e-4
                    rows[b][h] = {key: [r[key][i] for i in keep] for key in r}
        q, k, v = (f64(got[n]) for n in "qkv")
        attn = f64(got["attn"])
        for b in range(requests):
            keys, queries = turned(k[b], kw, rope, step), turned(q[b], qw, rope, step)
            for h in range(2):
                r = rows[b][h]
                r["k"].append(keys[h].astype(np.float16).astype(np.float64))
                r["v"].append(v[b, h].astype(np.float16).astype(np.float64))
                r["w"].append(0.0)
                score = queries[4 * h: 4 * h + 4] @ np.array(r["k"]).T / 8.0
                p = np.exp(score - score.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                want, size = p @ np.array(r["v"]), np.abs(r["v"]).max()
                # keys round to fp16 from fp32 here and from fp64 there: one unit of 2^-10 apart at most
                assert np.abs(attn[b, 4 * h: 4 * h + 4] - want).max() <= 2.0 ** -8 * size
                r["w"] = list(np.array(r["w"]) + p.sum(0))
                assert np.abs(f64(block.seen)[b, h, : len(r["w"])] - r["w"]).max() <= 2.0 ** -8 * len(r["w"])
        assert block.lens.tolist() == [len(rows[0][0]["w"])] * requests
    assert evicted == 4 and ops.get_error() == 0
    assert block.positions.tolist() == [60] * requests


@pytest.mark.gpu
def test_example_runs(cuda, monkeypatch, capsys):
    import paged_decode

    monkeypatch.setattr(sys, "argv", ["paged_decode.py", "--requests", "5", "--steps", "40", "--budget", "32",
                                      "--slack", "8"])
    paged_decode.main()
    said = capsys.readouterr().out
    assert "5 requests, 40 steps" in said and "1 evictions" in said


def test_example_needs_a_device():
    """There is no CPU path: the example fails loudly without CUDA."""
    if torch.cuda.is_available():
        pytest.skip("a device is here")
    from paged_decode import Block

    with pytest.raises((RuntimeError, AssertionError)):
        Block(1, hidden=256, q_heads=1, kv_heads=1, head_dim=64, fmt=packs.Q4K_RAW)
    assert paged.PAIRS == {"adjacent": 0, "halves": 1}
