"""Measured cases of the paged key-value cache operators.

Three operators share one cache of fixed-size pages:

* append: every query and key head is RMS-normalised, rotated by its token's position and
  rounded; keys and values go to their slots in the pages, queries to their own tensor;
* attend: one new token per sequence attends to its sequence's slots, optionally adding the
  attention weight that each slot received to a running sum;
* evict: each sequence and head keeps its first slots, its latest slots and, of the rest,
  those with the largest summed weight; kept rows move to the front of another set of pages.

`run` computes them in plain torch operations (`own` false) or with the package's kernels
(`own` true).  `exact` restates them in 64 bits.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

EPS = 1e-5
ROPE_BASE = 500000.0
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# --------------------------------------------------------------------------- cases

def _append(name, tokens, seqs, past, q_heads, kv_heads, dim, rot, src, cache, page, order,
            pairs, norm=True, pad=0):
    """`tokens` new rows over `seqs` sequences that hold `past` slots each; `pad` rows of
    the batch are padding; `order` is the order of heads and slots inside a page."""
    return dict(name=name, op="append", tokens=tokens, seqs=seqs, past=past, q_heads=q_heads,
                kv_heads=kv_heads, dim=dim, rot=rot, src=src, cache=cache, page=page,
                order=order, pairs=pairs, norm=norm, pad=pad)


def _attend(name, seqs, shortest, longest, q_heads, kv_heads, dim, src, cache, page, order,
            window=0, weights=False, empty=False):
    """One new token for each of `seqs` sequences of `shortest` to `longest` slots."""
    return dict(name=name, op="attend", seqs=seqs, shortest=shortest, longest=longest,
                q_heads=q_heads, kv_heads=kv_heads, dim=dim, src=src, cache=cache, page=page,
                order=order, window=window, weights=weights, empty=empty)


def _evict(name, seqs, shortest, longest, budget, sink, recent, kv_heads, dim, cache, page, order):
    return dict(name=name, op="evict", seqs=seqs, shortest=shortest, longest=longest,
                budget=budget, sink=sink, recent=recent, kv_heads=kv_heads, dim=dim,
                cache=cache, page=page, order=order)


def listed():
    return [
        # one decode step of a lone request, the heads of the 70B-class decoder: latency
        _append("append 1 token", 1, 1, 600, 64, 8, 128, 128, "f32", "f16", 16, "hsd", "adjacent"),
        # a decode step of a full batch, three rows of it padding
        _append("append 32 tokens", 32, 32, 300, 64, 8, 128, 128, "f32", "f16", 16, "hsd", "adjacent",
                pad=3),
        # a chunk of two prompts, pages ordered slot by slot, a partial rotation of odd width
        _append("append 2047 tokens", 2047, 2, 33, 32, 8, 80, 32, "bf16", "bf16", 24, "shd", "halves",
                pad=1),
        # the prompts of a busy server in one pass
        _append("append 16384 tokens", 16384, 8, 0, 64, 8, 128, 128, "bf16", "bf16", 64, "hsd", "halves"),
        # a lone request early in its answer: latency
        _attend("attend 1 x 511", 1, 511, 511, 64, 8, 128, "f32", "f16", 16, "hsd"),
        # a lone request with a very long context: all SMs work for a few heads
        _attend("attend 1 x 131072", 1, 131072, 131072, 64, 8, 128, "f32", "f16", 64, "hsd"),
        # a mixed batch that keeps the attention weights for later eviction, one request empty
        _attend("attend 32 x ..8191 weights", 32, 1, 8191, 32, 8, 128, "bf16", "bf16", 16, "shd",
                weights=True, empty=True),
        # as many key heads as query heads, small heads, a sliding window that starts inside a page
        _attend("attend 64 x ..4097 window", 64, 1000, 4097, 16, 16, 64, "f16", "f16", 24, "hsd",
                window=2000),
        # a full batch of long contexts: bandwidth
        _attend("attend 16 x 32768", 16, 32768, 32768, 64, 8, 128, "f16", "f16", 32, "hsd"),
        # a lone request goes back to its budget: latency
        _evict("evict 1 x 2500", 1, 2500, 2500, 2048, 4, 256, 8, 128, "f16", 16, "hsd"),
        # a ragged batch, some requests still below the budget
        _evict("evict 16 x ..9001", 16, 700, 9001, 1500, 4, 301, 8, 80, "bf16", 24, "shd"),
        # a batch of long contexts cut to a quarter
        _evict("evict 8 x 32768", 8, 32768, 32768, 8192, 16, 1024, 8, 128, "f16", 32, "hsd"),
    ]


HEADS = [(64, 8), (32, 8), (40, 8), (28, 4), (20, 4), (16, 16), (16, 1), (32, 1)]
DIMS = [(64, (16, 32, 64)), (80, (32, 80)), (112, (32, 64, 112)), (128, (32, 64, 128)), (256, (64, 128, 256))]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["append", "attend", "attend", "evict"])
    q_heads, kv_heads = rng.choice(HEADS)
    dim, rots = rng.choice(DIMS)
    cache = rng.choice(["f16", "bf16"])
    src = rng.choice(["f32", cache])
    page, order = rng.choice([8, 16, 24, 32, 64, 100, 128]), rng.choice(["hsd", "shd"])
    row = kv_heads * dim * 4  # bytes of one slot, keys and values
    if op == "append":
        tokens = spread(1, min(16384, 3e8 / ((q_heads + 2 * kv_heads) * dim * 4)))
        seqs = tokens if tokens <= 64 and rng.random() < 0.7 else rng.randint(1, min(tokens, 8))
        case = _append("", tokens, seqs, spread(1, 500), q_heads, kv_heads, dim, rng.choice(rots),
                       src, cache, page, order, rng.choice(["adjacent", "halves"]),
                       norm=rng.random() < 0.75, pad=rng.randint(0, min(4, tokens - 1)))
    elif op == "attend":
        seqs = spread(1, 128)
        longest = spread(1, min(131072, 8e8 / (row * seqs)))
        case = _attend("", seqs, spread(1, longest), longest, q_heads, kv_heads, dim, src, cache,
                       page, order, window=rng.choice([0, 0, spread(1, longest)]),
                       weights=rng.random() < 0.3, empty=seqs > 1 and rng.random() < 0.3)
    else:
        seqs = spread(1, 64)
        longest = spread(16, min(65536, 5e8 / (row * seqs)))
        budget = max(8, int(longest * rng.uniform(0.1, 0.9)))
        case = _evict("", seqs, spread(1, longest), longest, budget, rng.randint(0, 4),
                      rng.randint(0, budget // 2), kv_heads, dim, cache, page, order)
    del case["name"]
    return case


def _lengths(case):
    """The sequences' lengths, shortest to longest in equal ratios: their sum does not
    depend on the seed, only their order does."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    out = [int(round(lo * (hi / lo) ** (i / max(1, n - 1)))) for i in range(n)]
    out[-1] = hi
    if case.get("empty"):
        out[0] = 0
    return out


def _counts(case):
    """New tokens of each sequence of an append, padding rows left out."""
    live = case["tokens"] - case["pad"]
    return [live // case["seqs"] + (i < live % case["seqs"]) for i in range(case["seqs"])]


def work(case):
    e, row = BYTES[case["cache"]], 2 * case["kv_heads"] * case["dim"]
    if case["op"] == "append":
        t, live, d = case["tokens"], case["tokens"] - case["pad"], case["dim"]
        heads = case["q_heads"] + 2 * case["kv_heads"]
        read = live * heads * d * BYTES[case["src"]] + live * case["rot"] * 4 + t * 12
        return {"bytes": read + t * case["q_heads"] * d * BYTES[case["src"]] + live * row * e,
                "flops": live * (case["q_heads"] + case["kv_heads"]) * d * 7}
    lens = _lengths(case)
    if case["op"] == "attend":
        seen = sum(min(n, case["window"]) if case["window"] else n for n in lens)
        q = case["seqs"] * case["q_heads"] * case["dim"]
        kept = sum(lens) * case["kv_heads"] * 8 if case["weights"] else 0
        return {"bytes": seen * row * e + 2 * q * BYTES[case["src"]] + kept + case["seqs"] * case["q_heads"] * 4,
                "flops": 4 * seen * case["q_heads"] * case["dim"]}
    kept = sum(min(n, case["budget"]) for n in lens)
    heads, longest = case["kv_heads"], case["longest"]
    read = sum(n for n in lens if n > case["budget"]) * heads * 4
    return {"bytes": 2 * kept * row * e + read + case["seqs"] * heads * (4 * longest + 4 * case["budget"]),
            "flops": sum(lens) * heads}


# --------------------------------------------------------------------------- inputs

def _pages(case, capacity, gen, spare=0):
    """Key and value pools seen as [page, head, slot, dim], and each sequence's pages in an
    order of no pattern; `spare` slots more per sequence are a second set of pages."""
    dev, dt = gen.device, DTYPES[case["cache"]]
    per, extra = -(-max(capacity, 1) // case["page"]), -(-spare // case["page"])
    n, h, p, d = case["seqs"] * (per + extra) + 3, case["kv_heads"], case["page"], case["dim"]

    def pool():
        shape = (n, h, p, d) if case["order"] == "hsd" else (n, p, h, d)
        t = torch.empty(shape, dtype=dt, device=dev).normal_(generator=gen)
        return t if case["order"] == "hsd" else t.permute(0, 2, 1, 3)

    ids = torch.randperm(n, generator=gen, device=dev)[: case["seqs"] * (per + extra)].int()
    ids = ids.view(case["seqs"], per + extra)
    return pool(), pool(), ids[:, :per].contiguous(), ids[:, per:].contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    hq, hk, d = case["q_heads"] if "q_heads" in case else 0, case["kv_heads"], case["dim"]
    st = {"case": case}
    if case["op"] == "append":
        t, counts, past = case["tokens"], _counts(case), case["past"]
        st["k"], st["v"], st["table"], _ = _pages(case, past + max(counts), gen)
        # queries, keys and values side by side, as one projection leaves them
        qkv = torch.empty(t, (hq + 2 * hk) * d, device=dev).normal_(generator=gen).mul_(3).to(DTYPES[case["src"]])
        st["q_new"] = qkv[:, : hq * d].view(t, hq, d)
        st["k_new"] = qkv[:, hq * d: (hq + hk) * d].view(t, hk, d)
        st["v_new"] = qkv[:, (hq + hk) * d:].view(t, hk, d)
        n = torch.tensor(counts, device=dev)
        seqs = torch.repeat_interleave(torch.arange(case["seqs"], device=dev), n)
        at = torch.arange(t - case["pad"], device=dev) - (n.cumsum(0) - n)[seqs] + past
        none = torch.full((case["pad"],), -1, device=dev)
        st["seqs"] = torch.cat([seqs, none * 0]).int()
        st["slots"] = torch.cat([at, none]).int()
        st["positions"] = torch.cat([at + 7 * seqs, none]).int()  # positions run ahead of evicted slots
        angle = torch.arange(past + max(counts) + 7 * case["seqs"], device=dev, dtype=torch.float64)[:, None] * (
            ROPE_BASE ** (-torch.arange(0, case["rot"], 2, device=dev, dtype=torch.float64) / case["rot"]))
        st["rope"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        for w in ("q_norm", "k_norm"):
            st[w] = 1 + 0.1 * torch.randn(d, generator=gen, device=dev) if case["norm"] else None
        return st
    lens = torch.tensor(_lengths(case), device=dev)[torch.randperm(case["seqs"], generator=gen, device=dev)].int()
    st["lens"], longest = lens, case["longest"]
    st["k"], st["v"], st["table"], st["new_table"] = _pages(case, longest, gen, case.get("budget", 0))
    past_end = torch.arange(longest, device=dev) >= lens[:, None]
    if case["op"] == "attend":
        # whatever an earlier owner left in the slots past a sequence's end
        page, slot = _slots(st["table"], torch.arange(longest, device=dev).expand(case["seqs"], longest), case["page"])
        for pool in (st["k"], st["v"]):
            pool.permute(0, 2, 1, 3)[page[past_end], slot[past_end]] = math.nan
        st["q"] = torch.empty(case["seqs"], hq, d, device=dev).normal_(generator=gen).mul_(2).to(DTYPES[case["src"]])
    if case["op"] == "evict" or case["weights"]:
        # a few slots take most of the weight, some never had any
        w = torch.empty(case["seqs"], hk, longest, device=dev).normal_(generator=gen).mul_(2).exp_()
        w *= torch.rand(w.shape, generator=gen, device=dev) > 0.2
        st["weight"] = w.masked_fill_(past_end[:, None], 0.0)
        st["new_weight"] = torch.zeros_like(w)
    return st


def _slots(table, at, page):
    """Page and slot inside it of the logical slots at[sequence, ...]."""
    flat = at.reshape(at.shape[0], -1)
    return table.long().gather(1, flat // page).view(at.shape), at % page


# --------------------------------------------------------------------------- plain form

def _rows(pool, table, longest):
    """The pages of each sequence one after another: [sequence, head, slot, dim]."""
    s, h, d = table.shape[0], pool.shape[1], pool.shape[3]
    return pool[table.long()].permute(0, 2, 1, 3, 4).reshape(s, h, -1, d)[:, :, :longest]


def _turned(x, cos, sin, pairs):
    """x[..., :rot] with every pair turned by its angle; pairs are neighbours or half a width apart."""
    rot = 2 * cos.shape[-1]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs == "adjacent" else (x[..., : rot // 2], x[..., rot // 2: rot])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([a, b], -1).flatten(-2) if pairs == "adjacent" else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _plain_append(st):
    case = st["case"]
    live = st["positions"] >= 0
    half = case["rot"] // 2
    angles = st["rope"][st["positions"].clamp_min(0).long()][:, None]
    cos, sin = angles[..., :half], angles[..., half:]

    def head(x, w):
        x = x.float()
        if w is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        return _turned(x, cos, sin, case["pairs"])

    q = torch.where(live[:, None, None], head(st["q_new"], st["q_norm"]), 0.0).to(st["q_new"].dtype)
    k = head(st["k_new"], st["k_norm"]).to(st["k"].dtype)
    v = st["v_new"].float().to(st["v"].dtype)
    n = case["tokens"] - case["pad"]  # the padding rows are the last ones
    slot = st["slots"][:n].long()
    page = st["table"].long()[st["seqs"][:n].long(), slot // case["page"]]
    for pool, new in ((st["k"], k), (st["v"], v)):
        pool.permute(0, 2, 1, 3)[page, slot % case["page"]] = new[:n]
    return {"q": q, "k": st["k"], "v": st["v"]}


def _plain_attend(st):
    case = st["case"]
    s, hq, hk, d, longest = case["seqs"], case["q_heads"], case["kv_heads"], case["dim"], case["longest"]
    at = torch.arange(longest, device=st["q"].device)
    seen = at < st["lens"][:, None]
    if case["window"]:
        seen = seen & (at >= st["lens"][:, None] - case["window"])
    seen = seen[:, None, :, None]
    k = torch.where(seen, _rows(st["k"], st["table"], longest).float(), 0.0)
    v = torch.where(seen, _rows(st["v"], st["table"], longest).float(), 0.0)
    q = st["q"].float().view(s, hk, hq // hk, d) * d ** -0.5
    score = torch.where(seen.transpose(2, 3), torch.matmul(q, k.transpose(2, 3)), -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    share = 1.0 / torch.where(total > 0, total, 1.0)
    out = {"out": (torch.matmul(p, v) * share).view(s, hq, d).to(st["q"].dtype),
           "lse": (top + total.log()).view(s, hq)}
    if case["weights"]:
        st["new_weight"].copy_(st["weight"] + (p * share).sum(2))
        out["weight"] = st["new_weight"]
    return out


def _plain_evict(st):
    case = st["case"]
    s, h, budget, longest = case["seqs"], case["kv_heads"], case["budget"], case["longest"]
    lens = st["lens"].long()[:, None, None]
    at = torch.arange(longest, device=st["weight"].device).expand(s, h, longest)
    rank = torch.where(at < lens, st["weight"], -math.inf)
    always = (at < case["sink"]) | ((at >= lens - case["recent"]) & (at < lens))
    rank = torch.where(always, math.inf, rank)
    take = min(budget, longest)
    best = rank.sort(dim=-1, descending=True, stable=True).indices[..., :take]
    best = torch.where(torch.arange(take, device=at.device) < lens, best, longest)  # a short sequence has no more
    best = best.sort(-1).values
    kept = torch.nn.functional.pad(torch.where(best < longest, best, -1), (0, budget - take), value=-1)
    # entries without a slot repeat the first one's move
    i = torch.arange(budget, device=at.device).expand(s, h, budget)
    i = torch.where(kept >= 0, i, 0)
    from_ = torch.where(kept >= 0, kept, kept[..., :1])
    heads = torch.arange(h, device=at.device)[None, :, None]
    (sp, ss), (dp, ds) = _slots(st["table"], from_, case["page"]), _slots(st["new_table"], i, case["page"])
    for pool in (st["k"], st["v"]):
        pool[dp, heads, ds] = pool[sp, heads, ss]
    st["new_weight"].zero_().scatter_(2, i, st["weight"].gather(2, from_))
    return {"kept": kept.int(), "lens": st["lens"].clamp_max(budget), "weight": st["new_weight"],
            "k": st["k"], "v": st["v"]}


# --------------------------------------------------------------------------- the package's kernels

def _own_append(st):
    from qgemv_b200 import paged

    case = st["case"]
    if "cache" not in st:
        st["cache"] = paged.PagedCache(st["k"], st["v"], st["table"])
    q = paged.qk_norm_rope_append(
        st["cache"], st["q_new"], st["k_new"], st["v_new"], st["rope"], st["positions"],
        slots=st["slots"], seqs=st["seqs"], q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS,
        pairs=case["pairs"])
    return {"q": q, "k": st["k"], "v": st["v"]}


def _own_attend(st):
    from qgemv_b200 import paged

    case = st["case"]
    if "plan" not in st:
        cache = paged.PagedCache(st["k"], st["v"], st["table"])
        st["plan"] = paged.AttentionPlan(cache, case["q_heads"], max_len=case["longest"],
                                         weights=case["weights"])
    more = {"weight_in": st["weight"], "weight_out": st["new_weight"]} if case["weights"] else {}
    out, lse = paged.attend(st["plan"], st["q"], st["lens"], window=case["window"], return_lse=True, **more)
    got = {"out": out, "lse": lse}
    if case["weights"]:
        got["weight"] = st["new_weight"]
    return got


def _own_evict(st):
    from qgemv_b200 import paged

    case = st["case"]
    if "cache" not in st:
        st["cache"] = paged.PagedCache(st["k"], st["v"], st["table"])
    kept, lens = paged.evict(st["cache"], st["lens"], st["weight"], case["budget"], sink=case["sink"],
                             recent=case["recent"], new_table=st["new_table"],
                             weight_out=st["new_weight"])
    return {"kept": kept, "lens": lens, "weight": st["new_weight"], "k": st["k"], "v": st["v"]}


PLAIN = {"append": _plain_append, "attend": _plain_attend, "evict": _plain_evict}
OWN = {"append": _own_append, "attend": _own_attend, "evict": _own_evict}


def run(state):
    if not own:
        return PLAIN[state["case"]["op"]](state)
    package = str(Path.cwd() / "local-ai-gpu-acceleration_b200")
    if package not in sys.path:
        sys.path.insert(0, package)
    return OWN[state["case"]["op"]](state)


# --------------------------------------------------------------------------- 64 bits

def exact(case, seed):
    st = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](case, st)


def _exact_append(case, st):
    t, half = case["tokens"], case["rot"] // 2
    where = [torch.arange(half, device="cuda") * 2, torch.arange(half, device="cuda") * 2 + 1] \
        if case["pairs"] == "adjacent" else \
        [torch.arange(half, device="cuda"), torch.arange(half, device="cuda") + half]
    pos = st["positions"].long()
    turn = torch.complex(st["rope"][:, :half].double(), st["rope"][:, half:].double())[pos.clamp_min(0)][:, None]

    def head(x, w):
        x = x.double().clone()
        if w is not None:
            x = x / ((x ** 2).sum(-1, keepdim=True) / case["dim"] + EPS).sqrt() * w.double()
        z = torch.complex(x[..., where[0]], x[..., where[1]]) * turn
        x[..., where[0]], x[..., where[1]] = z.real, z.imag
        return x

    q, k = head(st["q_new"], st["q_norm"]), head(st["k_new"], st["k_norm"])
    q[pos < 0] = 0.0
    pools = {n: st[n].double() for n in ("k", "v")}
    live = (pos >= 0).nonzero()[:, 0]
    slot, seq = st["slots"].long()[live], st["seqs"].long()[live]
    page = st["table"].long()[seq, slot // case["page"]]
    for h in range(case["kv_heads"]):
        pools["k"][page, h, slot % case["page"]] = k[live, h]
        pools["v"][page, h, slot % case["page"]] = st["v_new"].double()[live, h]
    assert q.shape[0] == t
    return {"q": q, **pools}


def _exact_attend(case, st):
    s, hq, hk, d = case["seqs"], case["q_heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(s, hq, d, dtype=torch.float64, device="cuda")
    lse = torch.full((s, hq), -math.inf, dtype=torch.float64, device="cuda")
    weight = None
    if case["weights"]:
        weight = st["weight"].double().clone()
    for b, n in enumerate(st["lens"].tolist()):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        at = torch.arange(first, n, device="cuda")
        page, slot = st["table"][b].long()[at // case["page"]], at % case["page"]
        for h in range(hk):
            k, v = st["k"][page, h, slot].double(), st["v"][page, h, slot].double()
            mine = slice(h * (hq // hk), (h + 1) * (hq // hk))
            score = st["q"][b, mine].double() @ k.T / math.sqrt(d)
            lse[b, mine] = torch.logsumexp(score, -1)
            p = (score - lse[b, mine, None]).exp()
            out[b, mine] = p @ v
            if weight is not None:
                weight[b, h, first:n] += p.sum(0)
    return {"out": out, "lse": lse, **({"weight": weight} if weight is not None else {})}


def _exact_evict(case, st):
    s, h, budget = case["seqs"], case["kv_heads"], case["budget"]
    weight = torch.zeros(s, h, case["longest"], dtype=torch.float64, device="cuda")
    pools = {n: st[n].double() for n in ("k", "v")}
    old = {n: st[n] for n in ("k", "v")}
    at = torch.arange(budget, device="cuda")
    for b, n in enumerate(st["lens"].tolist()):
        for j in range(h):
            w = st["weight"][b, j, :n].double()
            order = torch.arange(n, device="cuda")
            if n > budget:
                first, last = min(case["sink"], n), n - case["recent"]
                middle = torch.argsort(-w[first:last], stable=True)[: budget - first - case["recent"]] + first
                order = torch.cat([order[:first], middle.sort().values, order[last:]])
            m = order.numel()
            weight[b, j, :m] = w[order]
            src = st["table"][b].long()[order // case["page"]], order % case["page"]
            dst = st["new_table"][b].long()[at[:m] // case["page"]], at[:m] % case["page"]
            for name in ("k", "v"):
                pools[name][dst[0], j, dst[1]] = old[name][src[0], j, src[1]].double()
    return {"kept": None, "lens": None, "weight": weight, **pools}
