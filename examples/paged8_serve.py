"""Serving one attention block over a paged key-value cache in 8 bits.

Prompts come in ragged chunks, answers token by token, both through the same calls: the batched
quantized projections (qg_gemm_batched), the norm and rotation of queries and keys with the
quantising append (qg_qk_norm_rope_append8), attention with a sliding window and first tokens that stay
visible (qg_paged_attn8), the output projection.  A request that is to be cut back by attention
weight moves to the 16-bit cache, which can evict: its rows are read back (qg_kv_read8) and
written there.

    python examples/paged8_serve.py --requests 8 --prompt 600 --steps 256
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "local-ai-gpu-acceleration_b200"))

from qgemv_b200 import ops, packs, paged, paged8  # noqa: E402


class Block8:
    """One attention block of synthetic weights and the 8-bit cache of `requests` requests of up to
    max_len tokens, called with up to max_tokens rows."""

    def __init__(self, requests: int, max_len: int, max_tokens: int, hidden: int = 4096, q_heads: int = 32,
                 kv_heads: int = 8, head_dim: int = 128, page_size: int = 64, block: int = 32, window: int = 0,
                 sink: int = 4, dtype=torch.bfloat16, fmt: int = packs.Q4K_RAW, seed: int = 0, device: str = "cuda"):
        self.requests, self.hidden, self.fmt, self.dtype = requests, hidden, fmt, dtype
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.window, self.sink = window, sink
        rows = dict(q=q_heads * head_dim, k=kv_heads * head_dim, v=kv_heads * head_dim)
        shapes = {n: (r, hidden) for n, r in rows.items()} | {"o": (hidden, q_heads * head_dim)}
        self.weights = {name: (*ops.to_device(packs.synthetic_pack(fmt, r, c, seed=seed * 10 + i), device), r, c)
                        for i, (name, (r, c)) in enumerate(shapes.items())}
        gen = torch.Generator(device=device)
        gen.manual_seed(seed)
        self.norm = 1 + 0.02 * torch.randn(hidden, generator=gen, device=device)
        self.q_norm = 1 + 0.02 * torch.randn(head_dim, generator=gen, device=device)
        self.k_norm = 1 + 0.02 * torch.randn(head_dim, generator=gen, device=device)
        self.rope = paged.rope_table(max_len, head_dim, device=device)
        pages = -(-max_len // page_size)
        self.cache = paged8.PagedCache8.empty(requests * pages, kv_heads, page_size, head_dim, requests, pages,
                                              block=block, device=device)
        self.cache.table.copy_(torch.randperm(requests * pages, generator=gen, device=device).view(requests, pages))
        self.plan = paged8.AttentionPlan8(self.cache, q_heads, max_tokens=max_tokens)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.device = device

    def project(self, name: str, x: torch.Tensor) -> torch.Tensor:
        """Rows of x through a quantized matrix, 32 at a time."""
        payload, meta, rows, cols = self.weights[name]
        return torch.cat([ops.gemm_batched(self.fmt, payload, meta, part.contiguous(), rows, cols) for part in x.split(32)])

    def run(self, x: torch.Tensor, counts: list[int] | None = None) -> dict:
        """New tokens x [rows, hidden]: counts[b] of request b, one after another, or one of every request.
        Returns the stages; "out" is the block's output."""
        offsets = None
        new = torch.ones_like(self.lens)
        if counts is not None:
            new = torch.tensor(counts, dtype=torch.int32, device=self.device)
            offsets = torch.nn.functional.pad(new.cumsum(0, dtype=torch.int32), (1, 0))
        h = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * self.norm
        q, k, v = (self.project(n, h).to(self.dtype).view(x.shape[0], -1, self.head_dim) for n in "qkv")
        seqs = torch.repeat_interleave(torch.arange(self.requests, device=self.device), new.long(), output_size=x.shape[0])
        first = torch.zeros_like(self.lens) if offsets is None else offsets[:-1]
        positions = self.lens[seqs] + (0 if offsets is None else torch.arange(x.shape[0], device=self.device).int() - first[seqs])
        self.lens += new
        rotated = paged8.qk_norm_rope_append(self.cache, q, k, v, self.rope, positions.int().contiguous(), self.lens,
                                             offsets=offsets, q_norm=self.q_norm, k_norm=self.k_norm)
        attn = paged8.attend(self.plan, rotated, self.lens, offsets=offsets, window=self.window, sink=self.sink)
        out = x + self.project("o", attn.float().flatten(1))
        return dict(q=q, k=k, v=v, rotated=rotated, attn=attn, positions=positions, out=out)

    def widened(self, length: int, dtype=torch.float16) -> paged.PagedCache:
        """The first `length` slots of every request (all have as many) in a 16-bit cache of their own."""
        starts = torch.zeros_like(self.lens)
        offsets = torch.arange(self.requests + 1, dtype=torch.int32, device=self.device) * length
        rows = paged8.read(self.cache, starts, offsets, self.requests * length, dtype=dtype)
        # one page a request: its rows as they were read
        pools = (t.view(self.requests, length, self.kv_heads, self.head_dim).transpose(1, 2) for t in rows)
        table = torch.arange(self.requests, dtype=torch.int32, device=self.device).view(-1, 1)
        return paged.PagedCache(*pools, table)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=600)
    ap.add_argument("--steps", type=int, default=256)
    ap.add_argument("--window", type=int, default=0)
    a = ap.parse_args()
    counts = [a.prompt - 7 * (b % 5) for b in range(a.requests)]
    block = Block8(a.requests, a.prompt + a.steps + 8, sum(counts), window=a.window)
    x = block.run(torch.randn(sum(counts), block.hidden, device="cuda"), counts)["out"]
    x = x[torch.tensor(counts).cumsum(0) - 1]  # every request's last token
    for step in range(a.steps + 8):
        if step == 8:  # the first steps load the library's kernels
            torch.cuda.synchronize()
            began = time.perf_counter()
        x = block.run(x)["out"]
        x = x / x.square().mean(-1, keepdim=True).sqrt()
    torch.cuda.synchronize()
    took = time.perf_counter() - began
    assert ops.get_error() == 0
    print(f"{a.requests} requests, prompts of up to {a.prompt} tokens, {a.steps} steps: {1e6 * took / a.steps:.0f} us a step, "
          f"lengths {block.lens.tolist()}")


if __name__ == "__main__":
    main()
