"""Batched decode of one attention block over a paged key-value cache that evicts.

Several requests of different lengths decode together: the batched quantized projections
(qg_gemm_batched), the norm and rotation of queries and keys with the append to their pages
(qg_qk_norm_rope_append), attention over the pages with the weight that every slot receives
(qg_paged_attn), the output projection, and, whenever a request has grown past its budget,
eviction back to it (qg_kv_evict).  Rotary positions keep counting while slots are reused, so
positions and slots are kept apart.

    python examples/paged_decode.py --requests 8 --steps 1024 --budget 512
"""

from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "local-ai-gpu-acceleration_b200"))

from qgemv_b200 import ops, packs, paged  # noqa: E402


class Block:
    """One attention block of synthetic weights and the paged cache of `requests` requests.

    Each request owns enough pages for budget + slack slots; eviction brings it back to the
    budget when the slack is used up, within its own pages."""

    def __init__(self, requests: int, hidden: int = 4096, q_heads: int = 32, kv_heads: int = 8,
                 head_dim: int = 128, budget: int = 512, slack: int = 64, page_size: int = 16,
                 sink: int = 4, recent: int | None = None, fmt: int = packs.Q4K_RAW, max_positions: int = 65536,
                 seed: int = 0, device: str = "cuda"):
        self.requests, self.hidden, self.fmt = requests, hidden, fmt
        self.q_heads, self.kv_heads, self.head_dim = q_heads, kv_heads, head_dim
        self.budget, self.limit, self.sink = budget, budget + slack, sink
        self.recent = budget // 8 if recent is None else recent
        rows = dict(q=q_heads * head_dim, k=kv_heads * head_dim, v=kv_heads * head_dim)
        shapes = {n: (r, hidden) for n, r in rows.items()} | {"o": (hidden, q_heads * head_dim)}
        self.weights, self.workspaces = {}, {}
        for i, (name, (r, c)) in enumerate(shapes.items()):
            pack = packs.synthetic_pack(fmt, r, c, seed=seed * 10 + i)
            self.weights[name] = (*ops.to_device(pack, device), r, c)
            self.workspaces[name] = torch.empty(ops.gemm_batched_workspace_bytes(fmt, requests, r, c),
                                                dtype=torch.uint8, device=device)
        gen = torch.Generator(device=device)
        gen.manual_seed(seed)
        self.norm = 1 + 0.02 * torch.randn(hidden, generator=gen, device=device)
        self.q_norm = 1 + 0.02 * torch.randn(head_dim, generator=gen, device=device)
        self.k_norm = 1 + 0.02 * torch.randn(head_dim, generator=gen, device=device)
        self.rope = paged.rope_table(max_positions, head_dim, device=device)
        pages = -(-self.limit // page_size)
        self.cache = paged.PagedCache.empty(requests * pages, kv_heads, page_size, head_dim, requests,
                                            pages, device=device)
        self.cache.table.copy_(torch.randperm(requests * pages, generator=gen, device=device).view(requests, pages))
        self.plan = paged.AttentionPlan(self.cache, q_heads, max_len=self.limit, weights=True)
        self.lens = torch.zeros(requests, dtype=torch.int32, device=device)
        self.positions = torch.zeros(requests, dtype=torch.int32, device=device)
        self.seen = torch.zeros(requests, kv_heads, self.limit, device=device)  # weight of every slot
        self.longest = 0  # upper bound of lens on the host: every step adds one

    def project(self, name: str, x: torch.Tensor) -> torch.Tensor:
        payload, meta, rows, cols = self.weights[name]
        return ops.gemm_batched(self.fmt, payload, meta, x, rows, cols, workspace=self.workspaces[name])

    def step(self, x: torch.Tensor) -> dict:
        """One token of every request: x [requests, hidden] -> its stages, "out" the block's
        output and "kept" the slots that an eviction before the token left (None without one)."""
        kept = self.evict() if self.longest == self.limit else None
        h = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-5) * self.norm
        q = self.project("q", h).view(-1, self.q_heads, self.head_dim)
        k = self.project("k", h).view(-1, self.kv_heads, self.head_dim)
        v = self.project("v", h).view(-1, self.kv_heads, self.head_dim)
        rotated = paged.qk_norm_rope_append(self.cache, q, k, v, self.rope, self.positions, slots=self.lens,
                                            q_norm=self.q_norm, k_norm=self.k_norm)
        self.lens += 1
        self.positions += 1
        self.longest += 1
        attn = paged.attend(self.plan, rotated, self.lens, weight_in=self.seen, weight_out=self.seen)
        out = x + self.project("o", attn.view(x.shape[0], -1))
        return dict(q=q, k=k, v=v, attn=attn, out=out, kept=kept)

    def evict(self) -> torch.Tensor:
        """Requests past the budget go back to it, keeping what was attended to most."""
        kept, _ = paged.evict(self.cache, self.lens, self.seen, self.budget, sink=self.sink, recent=self.recent)
        self.longest = self.budget
        return kept


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--requests", type=int, default=8)
    ap.add_argument("--steps", type=int, default=1024)
    ap.add_argument("--budget", type=int, default=512)
    ap.add_argument("--slack", type=int, default=64)
    a = ap.parse_args()
    block = Block(a.requests, budget=a.budget, slack=a.slack)
    x = torch.randn(a.requests, block.hidden, device="cuda")
    evictions = 0
    for step in range(a.steps + 8):
        if step == 8:  # the first steps load the library's kernels
            torch.cuda.synchronize()
            began = time.perf_counter()
        got = block.step(x)
        evictions += got["kept"] is not None
        x = got["out"] / got["out"].square().mean(-1, keepdim=True).sqrt()
    torch.cuda.synchronize()
    took = time.perf_counter() - began
    assert ops.get_error() == 0
    print(f"{a.requests} requests, {a.steps} steps: {1e6 * took / a.steps:.0f} us a step, "
          f"{a.requests * a.steps / took:.0f} tokens/s through the block, {evictions} evictions, "
          f"lengths {block.lens.tolist()}")


if __name__ == "__main__":
    main()
