"""The 8-bit cache's operators as a server uses them (examples/paged8_serve.py): ragged prompts, then chunks
and single tokens, each stage against 64-bit arithmetic on the stage before; rows read back into a 16-bit cache.

A key that the cache holds is within half an e4m3 step of the formula's (test_paged8_append.py), here
|x| 2^-4 and, below the normal range, 2^-10 of a scale that is at most 2^-7 of the block's largest value,
and what scales that grew later cost: 2^-9 of the scale."""

import sys

import numpy as np
import pytest
import torch

from conftest import REPO
from paged8_util import logical
from qgemv_b200 import ops, packs, paged, paged8
from test_paged8_attn import check
from test_paged_append import formula

sys.path.insert(0, str(REPO / "examples"))

f64 = lambda t: t.double().cpu().numpy()  # noqa: E731


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,window", [(torch.bfloat16, 0), (torch.float32, 0), (torch.float16, 50)])
def test_prompts_chunks_and_tokens_follow_64_bits(cuda, dtype, window):
    from paged8_serve import Block8

    block = Block8(3, 300, 260, hidden=512, q_heads=8, kv_heads=2, head_dim=64, page_size=32, block=16,
                   window=window, sink=3, dtype=dtype)
    rope, qw, kw = f64(block.rope), f64(block.q_norm), f64(block.k_norm)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)
    lens, keys, values = [0, 0, 0], [[] for _ in range(3)], [[] for _ in range(3)]
    for counts in ([200, 1, 59], None, [0, 40, 3], None, None, [5, 5, 5]):
        new = counts or [1, 1, 1]
        got = block.run(torch.randn(sum(new), 512, generator=gen, device="cuda"), counts)
        pos = got["positions"].cpu().numpy()
        want_q, size_q = formula(f64(got["q"]), qw, 1e-5, rope, pos, "adjacent")
        want_k, _ = formula(f64(got["k"]), kw, 1e-5, rope, pos, "adjacent")
        unit = torch.finfo(dtype).eps / 2
        assert np.all(np.abs(f64(got["rotated"]) - want_q) <= 2.0 ** -20 * size_q + 1.01 * unit * np.abs(want_q) + 2.0 ** -25)
        row = 0
        for b, n in enumerate(new):
            assert list(pos[row: row + n]) == list(range(lens[b], lens[b] + n))
            keys[b] += list(want_k[row: row + n])
            values[b] += list(f64(got["v"])[row: row + n])
            lens[b] += n
            row += n
            for name, rows in (("k", keys), ("v", values)):
                want = np.array(rows[b]).transpose(1, 0, 2)
                held = logical(block.cache, name, b, lens[b]).numpy()
                top = np.abs(want).max()
                assert np.all(np.abs(held - want) <= 2.0 ** -4 * np.abs(want) + 2.0 ** -15 * top)
        assert block.lens.tolist() == lens
        check(block.cache, got["rotated"], lens, new, got["attn"], None, window, 3)
    assert ops.get_error() == 0


@pytest.mark.gpu
def test_a_request_goes_on_in_16_bits(cuda):
    """Read back and attended to in the 16-bit cache: the same rows, so the same output to both kernels'
    tolerances (2^-18 and 2^-16 of the largest value, and scores to 2^-20 each)."""
    from paged8_serve import Block8

    block = Block8(2, 128, 192, hidden=512, q_heads=8, kv_heads=2, head_dim=64, dtype=torch.float32)
    got = block.run(torch.randn(192, 512, device="cuda"), [96, 96])
    cache = block.widened(96)
    for b in range(2):
        for name in "kv":
            assert torch.equal(getattr(cache, name)[b].double().cpu(), logical(block.cache, name, b, 96))
    q = got["rotated"][[95, 191]].contiguous()
    plan = paged.AttentionPlan(cache, 8, weights=True)
    seen = torch.zeros(2, 2, 96, device="cuda")
    wide = paged.attend(plan, q, block.lens, weight_out=seen)
    one = paged8.attend(paged8.AttentionPlan8(block.cache, 8), q, block.lens)
    top = cache.v.abs().max().item()
    ds = q.norm(dim=-1).max().item() * cache.k.float().norm(dim=-1).max().item() / 8 * 2.0 ** -20
    assert ((wide - one).abs() <= (4 * ds + 2.0 ** -15) * top).all()
    assert ((one - got["attn"][[95, 191]]).abs() <= (4 * ds + 2.0 ** -15) * top).all()
    kept, lens = paged.evict(cache, block.lens.clone(), seen, 32, sink=4, recent=8)
    assert lens.tolist() == [32, 32] and (kept[..., :4] == torch.arange(4, device="cuda")).all() and ops.get_error() == 0


@pytest.mark.gpu
def test_example_runs(cuda, monkeypatch, capsys):
    import paged8_serve

    monkeypatch.setattr(sys, "argv", ["paged8_serve.py", "--requests", "5", "--prompt", "70", "--steps", "12"])
    paged8_serve.main()
    assert "5 requests, prompts of up to 70 tokens, 12 steps" in capsys.readouterr().out


def test_example_needs_a_device():
    """There is no CPU path: the example fails loudly without CUDA."""
    if torch.cuda.is_available():
        pytest.skip("a device is here")
    from paged8_serve import Block8

    with pytest.raises((RuntimeError, AssertionError)):
        Block8(1, 64, 8, hidden=256, q_heads=1, kv_heads=1, head_dim=64, fmt=packs.Q4K_RAW)
