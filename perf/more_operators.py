"""Measured cases of the operators of a paged key-value cache held in 8 bits.

Keys and values are e4m3 codes; every block of `block` consecutive slots of a page and kv head
has one scale for its keys and one for its values, the least power of two that keeps the block's
values within e4m3's range.  Three operators share the cache:

* append: every new query and key head is RMS-normalised and rotated by its token's position,
  queries are rounded to their own tensor, keys and values quantised into their blocks; a block
  whose scale has to grow has the codes that it holds already scaled down;
* read: rows of the cache as the 16- or 32-bit values they stand for, sequence after sequence;
* attend: the new tokens of every sequence, one or many, attend to the slots up to their own, or
  to the last `window` of them and the first `sink`.

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
TOP = 448.0  # e4m3's largest value
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f32": 4, "f16": 2, "bf16": 2}


# --------------------------------------------------------------------------- cases

def _append(name, seqs, tokens, past, q_heads, kv_heads, dim, rot, src, page, block, order, pairs,
            norm=True, pad=0):
    """`tokens` new rows over `seqs` sequences that hold `past` to twice as many slots, or one row
    a sequence where `tokens` is 0; the last `pad` rows belong to no sequence."""
    return dict(name=name, op="append", seqs=seqs, tokens=tokens, past=past, q_heads=q_heads,
                kv_heads=kv_heads, dim=dim, rot=rot, src=src, page=page, block=block, order=order,
                pairs=pairs, norm=norm, pad=pad)


def _read(name, seqs, shortest, longest, kv_heads, dim, src, page, block, order):
    """Rows of `seqs` sequences, `shortest` to `longest` of each, from some slot on."""
    return dict(name=name, op="read", seqs=seqs, shortest=shortest, longest=longest,
                kv_heads=kv_heads, dim=dim, src=src, page=page, block=block, order=order)


def _attend(name, seqs, shortest, longest, fresh, q_heads, kv_heads, dim, src, page, block, order,
            window=0, sink=0, empty=False):
    """`seqs` sequences of `shortest` to `longest` slots; the last `fresh` slots of the longest,
    and the same share of the others, are new tokens, or one of each where `fresh` is 0."""
    return dict(name=name, op="attend", seqs=seqs, shortest=shortest, longest=longest, fresh=fresh,
                q_heads=q_heads, kv_heads=kv_heads, dim=dim, src=src, page=page, block=block,
                order=order, window=window, sink=sink, empty=empty)


def listed():
    return [
        # a decode step of a batch with three rows of padding: latency, scales that grow
        _append("append8 32 tokens", 32, 0, 300, 64, 8, 128, 128, "f32", 32, 32, "hsd", "adjacent", pad=3),
        # a chunk of two prompts that starts inside a block, a partial rotation of odd width
        _append("append8 2047 tokens", 2, 2047, 33, 32, 8, 80, 32, "bf16", 48, 16, "shd", "halves", pad=1),
        # the prompts of a busy server in one pass
        _append("append8 16384 tokens", 8, 16384, 0, 64, 8, 128, 128, "bf16", 64, 64, "hsd", "halves"),
        # the rows of one short request, for another cache: latency
        _read("read8 1 x 700", 1, 700, 700, 8, 128, "f32", 32, 32, "hsd"),
        # a batch of long contexts: bandwidth
        _read("read8 8 x ..30001", 8, 9000, 30001, 8, 128, "f16", 64, 32, "shd"),
        # a lone request early in its answer: latency
        _attend("attend8 1 x 511", 1, 511, 511, 0, 64, 8, 128, "f32", 32, 32, "hsd"),
        # a lone request with a very long context: all SMs work for a few heads
        _attend("attend8 1 x 131072", 1, 131072, 131072, 0, 64, 8, 128, "f32", 64, 64, "hsd"),
        # as many key heads as query heads, small heads, a window that starts inside a block and
        # first tokens that stay visible, one request empty
        _attend("attend8 64 x ..4097 window", 64, 1000, 4097, 0, 16, 16, 64, "f16", 48, 16, "shd",
                window=2000, sink=5, empty=True),
        # a full batch of long contexts: bandwidth
        _attend("attend8 16 x 32768", 16, 32768, 32768, 0, 64, 8, 128, "f16", 32, 32, "hsd"),
        # a few drafted tokens of every request are checked at once
        _attend("attend8 16 x 5 of ..3000", 16, 200, 3000, 5, 32, 8, 128, "f32", 32, 32, "hsd"),
        # ragged prompts with a sliding window and first tokens that stay visible
        _attend("attend8 4 x ..2600 window", 4, 300, 2600, 2501, 32, 8, 64, "f16", 64, 32, "hsd",
                window=1000, sink=4),
        # the second chunk of a long prompt: matrix products
        _attend("attend8 4096 of 5600", 1, 5600, 5600, 4096, 64, 8, 128, "bf16", 64, 64, "hsd"),
    ]


HEADS = [(64, 8), (32, 8), (40, 8), (28, 4), (20, 4), (16, 16), (16, 1), (32, 1)]
DIMS = [(64, (16, 32, 64)), (80, (32, 80)), (112, (32, 64, 112)), (128, (32, 64, 128)), (256, (64, 128, 256))]
PAGES = [(16, 16), (32, 16), (32, 32), (48, 16), (64, 32), (64, 64), (96, 32), (128, 128), (128, 32)]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    op = rng.choice(["append", "read", "attend", "attend", "attend"])
    q_heads, kv_heads = rng.choice(HEADS)
    dim, rots = rng.choice(DIMS)
    src = rng.choice(["f32", "f16", "bf16"])
    page, block = rng.choice(PAGES)
    order = rng.choice(["hsd", "shd"])
    row = kv_heads * dim * 2  # bytes of one slot, keys and values
    if op == "append":
        if rng.random() < 0.4:
            seqs = spread(1, 256)
            case = _append("", seqs, 0, spread(1, min(2000, 1e8 / (row * seqs))), q_heads, kv_heads, dim,
                           rng.choice(rots), src, page, block, order, rng.choice(["adjacent", "halves"]),
                           norm=rng.random() < 0.75, pad=rng.randint(0, min(4, seqs - 1)))
        else:
            tokens = spread(1, min(16384, 3e8 / ((q_heads + 2 * kv_heads) * dim * 4)))
            seqs = rng.randint(1, min(tokens, 12))
            case = _append("", seqs, tokens, spread(1, 500), q_heads, kv_heads, dim, rng.choice(rots), src,
                           page, block, order, rng.choice(["adjacent", "halves"]), norm=rng.random() < 0.75,
                           pad=rng.randint(0, min(4, tokens - seqs)))
    elif op == "read":
        seqs = spread(1, 64)
        longest = spread(1, min(65536, 3e8 / (row * seqs)))
        case = _read("", seqs, spread(1, longest), longest, kv_heads, dim, src, page, block, order)
    else:
        many = rng.random() < 0.5
        seqs = spread(1, 16 if many else 128)
        longest = spread(1, min(131072, 8e8 / (row * seqs)))
        fresh = 0
        if many:  # at most about the products, and the scores in memory, of the largest listed case
            longest = min(longest, 12000)
            most = min(4e11 / (4 * seqs * longest * q_heads * dim), 4e9 / (4 * seqs * longest * q_heads))
            fresh = spread(1, min(longest, max(1, most)))
        case = _attend("", seqs, spread(1, longest), longest, fresh, q_heads, kv_heads, dim, src, page,
                       block, order, window=rng.choice([0, 0, spread(1, longest)]),
                       sink=rng.choice([0, rng.randint(1, 40)]), empty=seqs > 1 and rng.random() < 0.3)
    del case["name"]
    return case


def _lengths(case):
    """The sequences' lengths, shortest to longest in equal ratios."""
    n, lo, hi = case["seqs"], case["shortest"], case["longest"]
    out = [int(round(lo * (hi / lo) ** (i / max(1, n - 1)))) for i in range(n)]
    out[-1] = hi
    if case.get("empty"):
        out[0] = 0
    return out


def _fresh(case, length):
    """New tokens of an attending sequence."""
    if case["fresh"] == 0:
        return min(length, 1)
    return min(length, max(1, length * case["fresh"] // case["longest"]))


def _appended(case):
    """Slots that every sequence of an append holds already, and its new tokens."""
    n, past = case["seqs"], case["past"]
    before = [past + past * i // n for i in range(n)]
    if case["tokens"] == 0:
        return before, [int(i < n - case["pad"]) for i in range(n)]
    live = case["tokens"] - case["pad"]
    return before, [live // n + (i < live % n) for i in range(n)]


def work(case):
    h, d = case["kv_heads"], case["dim"]
    slot = 2 * h * d * (1 + 4 / (case["block"] * d))  # codes and scales of a slot
    if case["op"] == "append":
        before, new = _appended(case)
        live, b = sum(new), case["block"]
        rows = case["tokens"] or case["seqs"]
        heads = case["q_heads"] + 2 * h
        read = live * heads * d * BYTES[case["src"]] + live * case["rot"] * 4 + rows * 12
        kept = sum(8 * h for p, n in zip(before, new) if n and p % b)  # scales of blocks that were begun
        return {"bytes": read + live * case["q_heads"] * d * BYTES[case["src"]] + live * slot + kept,
                "flops": live * (case["q_heads"] + 2 * h) * d * 8}
    lens = _lengths(case)
    if case["op"] == "read":
        return {"bytes": sum(lens) * (slot + 2 * h * d * BYTES[case["src"]]), "flops": sum(lens) * 2 * h * d}
    w, sink, hq = case["window"], case["sink"], case["q_heads"]
    seen = pairs = rows = 0
    for n in lens:
        new = _fresh(case, n)
        rows += new
        first = n - new  # slot of the first new token
        if w:
            # slots of any new token's window, and the first ones
            low = max(0, first + 1 - w)
            seen += n - low + min(sink, low)
            pairs += sum(min(p + 1, w) + min(sink, max(0, p + 1 - w)) for p in range(first, n))
        else:
            seen += n
            pairs += new * (first + n + 1) // 2
    return {"bytes": seen * slot + 2 * rows * hq * d * BYTES[case["src"]] + rows * hq * 4,
            "flops": 4 * pairs * hq * d}


# --------------------------------------------------------------------------- inputs

def _pools(case, capacity, gen):
    """Codes and scales of keys and values seen as [page, head, slot, dim] and [page, head, block],
    as quantising values of several sizes leaves them, and each sequence's pages in an order of
    no pattern."""
    dev, page, block = gen.device, case["page"], case["block"]
    per = -(-max(capacity, 1) // page)
    n, h, d = case["seqs"] * per + 3, case["kv_heads"], case["dim"]

    def pool():
        x = torch.empty(n, h, page // block, block, d, device=dev).normal_(generator=gen)
        x *= torch.empty(n, h, page // block, 1, 1, device=dev).normal_(generator=gen).mul_(0.7).exp_()
        power = torch.frexp(x.abs().amax((-1, -2)) / TOP).exponent
        scale = torch.pow(2.0, power.double()).float()
        x /= scale[..., None, None]
        codes = x.view(n, h, page, d).to(torch.float8_e4m3fn).view(torch.uint8)
        if case["order"] == "shd":
            codes = codes.transpose(1, 2).contiguous().transpose(1, 2)
        return codes.view(torch.float8_e4m3fn), scale

    k, k_scale = pool()
    v, v_scale = pool()
    table = torch.randperm(n, generator=gen, device=dev)[: case["seqs"] * per].int().view(case["seqs"], per)
    return dict(k=k, v=v, k_scale=k_scale, v_scale=v_scale, table=table)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(counts):
    out = [0]
    for n in counts:
        out.append(out[-1] + n)
    return out


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    hq, hk, d = case.get("q_heads", 0), case["kv_heads"], case["dim"]
    st = {"case": case}
    if case["op"] == "append":
        before, new = _appended(case)
        t = case["tokens"] or case["seqs"]
        lens = [p + n if n else 0 for p, n in zip(before, new)]
        st |= _pools(case, max(lens), gen)
        # queries, keys and values side by side, as one projection leaves them
        qkv = torch.empty(t, (hq + 2 * hk) * d, device=dev).normal_(generator=gen).mul_(3)
        qkv[:, hq * d:].view(t, 2 * hk, d).mul_(torch.rand(t, 2 * hk, 1, generator=gen, device=dev).add_(0.2))
        qkv = qkv.to(DTYPES[case["src"]])
        st["q_new"] = qkv[:, : hq * d].view(t, hq, d)
        st["k_new"] = qkv[:, hq * d: (hq + hk) * d].view(t, hk, d)
        st["v_new"] = qkv[:, (hq + hk) * d:].view(t, hk, d)
        st["lens"] = _ints(lens)
        st["offsets"] = _ints(_offsets(new)) if case["tokens"] else None
        where = [p + 7 * b + i for b, (p, n) in enumerate(zip(before, new)) for i in range(n)]
        st["positions"] = _ints(where + [-1] * case["pad"])  # positions run ahead of the slots
        angle = torch.arange(max(where) + 1, device=dev, dtype=torch.float64)[:, None] * (
            ROPE_BASE ** (-torch.arange(0, case["rot"], 2, device=dev, dtype=torch.float64) / case["rot"]))
        st["rope"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        for w in ("q_norm", "k_norm"):
            st[w] = 1 + 0.1 * torch.randn(d, generator=gen, device=dev) if case["norm"] else None
        return st
    lens = [_lengths(case)[i] for i in torch.randperm(case["seqs"], generator=gen, device=dev).tolist()]
    longest = case["longest"]
    if case["op"] == "read":
        starts = [(11 * b) % 50 for b in range(case["seqs"])]
        st |= _pools(case, max(s + n for s, n in zip(starts, lens)), gen)
        st["starts"], st["offsets"], st["rows"] = _ints(starts), _ints(_offsets(lens)), sum(lens)
        return st
    st |= _pools(case, longest, gen)
    st["lens"] = _ints(lens)
    # whatever an earlier owner left in the slots past a sequence's end, and in their scales
    at = torch.arange(longest, device=dev).expand(case["seqs"], longest)
    past = at >= st["lens"][:, None]
    page, slot = _places(st["table"], at, case["page"])
    per = case["page"] // case["block"]
    whole = past & (at % case["block"] == 0)
    for name in ("k", "v"):
        st[name].view(torch.uint8).permute(0, 2, 1, 3)[page[past], slot[past]] = 0x7F
        st[name + "_scale"].permute(0, 2, 1)[page[whole], (slot[whole] // case["block"]).clamp_max(per - 1)] = math.nan
    new = [_fresh(case, n) for n in lens]
    st["offsets"] = _ints(_offsets(new)) if case["fresh"] else None
    rows = sum(new) if case["fresh"] else case["seqs"]
    q = torch.empty(rows, hq, d, device=dev).normal_(generator=gen).mul_(2)
    st["q"], st["most"], st["rows"] = q.to(DTYPES[case["src"]]), max(new), rows
    return st


def _places(table, at, page):
    """Page and place inside it of the slots at[sequence, ...]."""
    flat = at.reshape(at.shape[0], -1)
    return table.long().gather(1, flat // page).view(at.shape), at % page


# --------------------------------------------------------------------------- plain form

def _power(top):
    """The least power of two, between 2^-60 and 2^60, whose product with e4m3's largest value is `top` or more."""
    part, exponent = torch.frexp(top)
    e = torch.where(part <= 0.875, exponent - 9, exponent - 8)
    e = torch.where(top > 0, e.clamp(-60, 60), -60)
    return ((e.int() + 127) << 23).view(torch.float32)


def _codes(x):
    """fp32 values as the bytes of the nearest e4m3 codes."""
    return x.clamp(-TOP, TOP).to(torch.float8_e4m3fn).view(torch.uint8)


def _values(codes):
    return codes.contiguous().view(torch.float8_e4m3fn).float()


def _turned(x, cos, sin, pairs):
    """x[..., :rot] with every pair turned by its angle; pairs are neighbours or half a width apart."""
    rot = 2 * cos.shape[-1]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if pairs == "adjacent" else (x[..., : rot // 2], x[..., rot // 2: rot])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([a, b], -1).flatten(-2) if pairs == "adjacent" else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., rot:]], -1)


def _rows_of(st):
    """Sequence and place in it of every row that a sequence has (the rows of a call are sequence
    after sequence)."""
    case = st["case"]
    if st["offsets"] is None:
        seq = torch.arange(case["seqs"], device=st["lens"].device)
        return seq, torch.zeros_like(seq), torch.ones_like(seq)
    rows = torch.arange(st["q"].shape[0] if "q" in st else case["tokens"] - case["pad"], device=st["lens"].device)
    off = st["offsets"].long()
    seq = torch.searchsorted(off[1:].contiguous(), rows, right=True)
    return seq, rows - off[seq], off[1:] - off[:-1]


def _plain_append(st):
    case = st["case"]
    page, block, hk = case["page"], case["block"], case["kv_heads"]
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
    n = (case["tokens"] or case["seqs"]) - case["pad"]  # the rows of no sequence are the last ones
    seq, place, counts = _rows_of(st)
    seq, place = seq[:n], place[:n]
    slot = st["lens"].long()[seq] - counts[seq] + place
    ids, at = st["table"].long()[seq, slot // page], slot % page
    # the block of every sequence's first new token holds what the sequence had there
    s = case["seqs"] - (case["pad"] if case["tokens"] == 0 else 0)
    first = st["lens"].long()[:s] - counts[:s]
    first_id, first_at = st["table"].long()[torch.arange(s, device=first.device), first // page], first % page // block
    begun = (first % block != 0)[:, None]
    in_block = first_at[:, None] * block + torch.arange(block, device=first.device)
    for name, new in (("k", head(st["k_new"], st["k_norm"])), ("v", st["v_new"].float())):
        new = new[:n]
        scale, codes = st[name + "_scale"], st[name].view(torch.uint8).permute(0, 2, 1, 3)
        blocks = ids * (page // block) + at // block
        top = torch.zeros(scale.shape[0] * scale.shape[2], hk, device=new.device)
        top.index_reduce_(0, blocks, new.abs().amax(-1), "amax")
        top = top.view(scale.shape[0], -1, hk).transpose(1, 2)
        grown = _power(top)
        old = torch.where(begun, scale[first_id, :, first_at], 0.0)
        to = torch.maximum(grown[first_id, :, first_at], old)
        held = codes[first_id[:, None], in_block]
        shrunk = _codes(_values(held) * (old / to)[:, None, :, None])
        codes[first_id[:, None], in_block] = torch.where(begun[..., None, None], shrunk, held)
        grown[first_id, :, first_at] = to
        scale[ids, :, at // block] = grown[ids, :, at // block]
        codes[ids, at] = _codes(new / grown[ids, :, at // block][..., None])
    return {"q": q, "k": st["k"], "v": st["v"], "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _plain_read(st):
    case = st["case"]
    rows = torch.arange(st["rows"], device=st["offsets"].device)
    off = st["offsets"].long()
    seq = torch.searchsorted(off[1:].contiguous(), rows, right=True)
    slot = st["starts"].long()[seq] + rows - off[seq]
    ids, at = st["table"].long()[seq, slot // case["page"]], slot % case["page"]
    out = {}
    for name in ("k", "v"):
        codes = st[name].view(torch.uint8).permute(0, 2, 1, 3)[ids, at]
        scale = st[name + "_scale"][ids, :, at // case["block"]]
        out[name] = (_values(codes) * scale[..., None]).to(DTYPES[case["src"]])
    return out


def _gathered(st, name, longest, seen):
    """Rows of every sequence, zero where no token sees them: [sequence, head, slot, dim]."""
    case, table = st["case"], st["table"].long()
    s, h, d = case["seqs"], case["kv_heads"], case["dim"]
    codes = _values(st[name].view(torch.uint8)[table]).unflatten(3, (-1, case["block"]))
    x = codes * st[name + "_scale"][table][..., None, None]
    x = x.flatten(3, 4).permute(0, 2, 1, 3, 4).reshape(s, h, -1, d)[:, :, :longest]
    return torch.where(seen, x, 0.0)


def _plain_attend(st):
    case = st["case"]
    s, hq, hk, d, longest, most = (case["seqs"], case["q_heads"], case["kv_heads"], case["dim"], case["longest"],
                                   st["most"])
    seq, place, counts = _rows_of(st)
    dev = st["q"].device
    lens = st["lens"].long()
    at = torch.arange(longest, device=dev)
    q = torch.zeros(s, most, hq, d, device=dev)
    q[seq, place] = st["q"].float() * d ** -0.5
    q = q.view(s, most, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(s, hk, -1, d)
    slot = (lens - counts)[:, None] + torch.arange(most, device=dev)  # of every new token
    last = torch.minimum(slot, lens[:, None] - 1)[..., None]
    seen = at <= last
    if case["window"]:
        seen &= (at > slot[..., None] - case["window"]) | (at < case["sink"])
    rows = (at < lens[:, None])[:, None, :, None]
    k, v = (_gathered(st, name, longest, rows) for name in ("k", "v"))
    seen = seen[:, None, None].expand(s, 1, hq // hk, most, longest).reshape(s, 1, -1, longest)
    score = torch.matmul(q, k.transpose(2, 3)).masked_fill_(~seen, -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(score.sub_(top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total > 0, total, 1.0)
    lse = (top + total.log()).view(s, hk, hq // hk, most)
    out = out.view(s, hk, hq // hk, most, d).permute(0, 3, 1, 2, 4).reshape(s, most, hq, d)
    lse = lse.permute(0, 3, 1, 2).reshape(s, most, hq)
    return {"out": out[seq, place].to(st["q"].dtype), "lse": lse[seq, place]}


# --------------------------------------------------------------------------- the package's kernels

def _cache(st):
    from qgemv_b200 import paged8

    if "cache" not in st:
        st["cache"] = paged8.PagedCache8(st["k"], st["v"], st["k_scale"], st["v_scale"], st["table"])
    return paged8, st["cache"]


def _own_append(st):
    paged8, cache = _cache(st)
    if "q_out" not in st:  # rows of no sequence are left as they are
        st["q_out"] = torch.zeros_like(st["q_new"], memory_format=torch.contiguous_format)
    q = paged8.qk_norm_rope_append(
        cache, st["q_new"], st["k_new"], st["v_new"], st["rope"], st["positions"], st["lens"],
        offsets=st["offsets"], q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS, pairs=st["case"]["pairs"],
        q_out=st["q_out"])
    return {"q": q, "k": st["k"], "v": st["v"], "k_scale": st["k_scale"], "v_scale": st["v_scale"]}


def _own_read(st):
    paged8, cache = _cache(st)
    k, v = paged8.read(cache, st["starts"], st["offsets"], st["rows"], dtype=DTYPES[st["case"]["src"]])
    return {"k": k, "v": v}


def _own_attend(st):
    paged8, cache = _cache(st)
    case = st["case"]
    if "plan" not in st:
        st["plan"] = paged8.AttentionPlan8(cache, case["q_heads"], max_tokens=st["rows"])
    out, lse = paged8.attend(st["plan"], st["q"], st["lens"], offsets=st["offsets"], window=case["window"],
                             sink=case["sink"], return_lse=True)
    return {"out": out, "lse": lse}


PLAIN = {"append": _plain_append, "read": _plain_read, "attend": _plain_attend}
OWN = {"append": _own_append, "read": _own_read, "attend": _own_attend}


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
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend}[case["op"]](case, st)


def _e4m3(x):
    """The nearest e4m3 values of float64 values, ties to the even mantissa, past the range its end."""
    size = x.abs().clamp(2.0 ** -6, TOP)
    step = torch.exp2(torch.floor(torch.log2(size)) - 3)
    return (torch.round(x / step) * step).clamp(-TOP, TOP)


def _exact_append(case, st):
    half, page, block = case["rot"] // 2, case["page"], case["block"]
    before, new = _appended(case)
    width = torch.arange(half, device="cuda")
    where = (2 * width, 2 * width + 1) if case["pairs"] == "adjacent" else (width, width + half)
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
    out = {"q": q}
    for name, rows in (("k", k), ("v", st["v_new"].double())):
        pool, scale = st[name].double(), st[name + "_scale"].double()
        row = 0
        for b, (p, n) in enumerate(zip(before, new)):
            slot = p
            while slot < p + n:  # block after block
                id_, at = st["table"][b, slot // page].long(), slot % page
                fill = min(block - at % block, p + n - slot)
                x, base = rows[row: row + fill].transpose(0, 1), at // block * block
                need = torch.exp2(torch.ceil(torch.log2(x.abs().amax((1, 2)) / TOP)))
                need = need.clamp(2.0 ** -60, 2.0 ** 60)
                if at % block:
                    need = torch.maximum(need, scale[id_, :, at // block])
                    held = pool[id_, :, base: base + block] * (scale[id_, :, at // block] / need)[:, None, None]
                    pool[id_, :, base: base + block] = _e4m3(held)
                scale[id_, :, at // block] = need
                pool[id_, :, at: at + fill] = _e4m3(x / need[:, None, None])
                slot, row = slot + fill, row + fill
        out[name], out[name + "_scale"] = pool, scale
    return out


def _exact_read(case, st):
    offsets, starts = st["offsets"].tolist(), st["starts"].tolist()
    out = {}
    for name in ("k", "v"):
        rows = []
        for b in range(case["seqs"]):
            at = torch.arange(starts[b], starts[b] + offsets[b + 1] - offsets[b], device="cuda")
            id_, place = st["table"][b].long()[at // case["page"]], at % case["page"]
            scale = st[name + "_scale"].double()[id_, :, place // case["block"]]
            rows.append(st[name].view(torch.uint8)[id_, :, place].view(torch.float8_e4m3fn).double() * scale[..., None])
        out[name] = torch.cat(rows)
    return out


def _exact_attend(case, st):
    hq, hk, d = case["q_heads"], case["kv_heads"], case["dim"]
    group = hq // hk
    out = torch.zeros(st["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(st["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    row = 0
    for b, n in enumerate(st["lens"].tolist()):
        new = _fresh(case, n)
        mine = slice(row, row + new)
        row += new if case["fresh"] else 1
        if n == 0:
            continue
        at = torch.arange(n, device="cuda")
        id_, place = st["table"][b].long()[at // case["page"]], at % case["page"]
        token = torch.arange(n - new, n, device="cuda")[:, None]
        seen = at <= token
        if case["window"]:
            seen &= (token - at < case["window"]) | (at < case["sink"])
        for h in range(hk):
            k, v = (st[x].view(torch.uint8)[id_, h, place].view(torch.float8_e4m3fn).double()
                    * st[x + "_scale"].double()[id_, h, place // case["block"]][:, None] for x in "kv")
            for g in range(h * group, (h + 1) * group):
                score = (st["q"][mine, g].double() @ k.T / math.sqrt(d)).masked_fill(~seen, -math.inf)
                lse[mine, g] = torch.logsumexp(score, -1)
                out[mine, g] = torch.softmax(score, -1) @ v
    return {"out": out, "lse": lse}
