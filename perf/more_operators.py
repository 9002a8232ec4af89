"""What a server does around a key/value cache held in 4 bits, as it is timed: where new tokens go, a chunk's attention
over the cache, and single tokens' attention over the pages that a cheap score selects.

A case is a dict of plain values.  ``kind`` says what one pass runs:

* ``append``: ``kv4_append``, room for a batch's new tokens: pages from a list of free ones into the page table, the
  tokens' slots and positions, row offsets, new lengths.  Functional but for the page table.
* ``chunk``: ``kv4_chunk_attention``, packed rows of new tokens (already stored) over their sequences' pages, causal: a
  sequence's last row sees all its tokens, the row before one fewer.
* ``summarize``: ``kv4_summarize``, the mean key of every page that new tokens went to, in 8 bits.  The summary comes
  back as the values it stands for.
* ``sparse``: ``kv4_select``, the ``count`` pages per sequence and key/value head whose mean keys promise the largest
  logits, then ``kv4_attention`` over a page table per key/value head.

The cache is uint8 [pages, key/value heads, page / 16, record]; a record holds 16 tokens of one head, D channels in
G = D / group groups for the keys and one group for the values:

    keys     16 tokens x D / 8 words; word (channel / 8) % 4 * (D / 32) + channel / 32 of a token
    (scale, minimum) of the keys     G x 16 tokens, float16 pairs
    values   D / 8 words x 16 tokens; word channel / 8
    (scale, minimum) of the values   16 tokens, float16 pairs

Channel c of a word's 8 is its nibble c / 2 + 4 * (c % 2); a code stands for minimum + scale * code.

The summary is int8 [pages, key/value heads, D + 16]: D codes, their float32 step (4 bytes), 12 unused ones.  With m the
mean of a page's keys (64 bits: exact sums) and 2^E <= max |m| < 2^(E + 1): step = 2^(E - 6), code = round(m / step)
within +-127 (a page of zeros: step 0).  Queries get codes the same way, one step per head.  The score of a page is
max over the group's heads of step(head) / max step * codes(head).codes(page) * step(page), the first factor at least
2^-40: whole numbers times powers of two, so that no sum is rounded and the selection is the same in any order of
summation.  The first and the last page are always selected, ties go to the lowest page, and the selected ones stand
in ascending order (-1 behind them).

Head counts, head sizes and lengths are those of bench.py's models (Llama-3-8B: 32 query and 8 key/value heads of 128
channels, Llama-3-70B: 64 and 8; prompts of 512 tokens at batch 32) and generic ones.  Queries, keys and values are
N(0, 1); keys have a per-channel offset of +-6 in 3 % of their channels and a part that stays the same through a page.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
LIMIT = 65504.0
# the largest listed cases: a sparse batch's cached bytes, a chunk's products
MOST_CACHED = 64 * 8192 * 8 * 2176 // 16
MOST_SCORES = 32 * 2048 * 32768


def _case(name, kind, dtype, heads, kv_heads, head, seqs, low, high, new=1, lead=0, page=16, group=0, width=0, count=0):
    """low..high: tokens of the shortest and the longest sequence before the new ones; new: new tokens of every
    sequence, lead: of the first one instead; width: of the page table (append); count: selected pages"""
    c = {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head": head, "seqs": seqs, "low": low,
         "high": high, "new": new, "lead": lead or new, "page": page, "group": group or head, "width": width,
         "count": count}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one decode step of the benchmark's batch: latency
        _case("append_32x1", "append", "f16", 32, 8, 128, 32, 512, 640, width=64),
        # many sequences that get a chunk of their prompts each, wide page table
        _case("append_256x33", "append", "f16", 32, 8, 128, 256, 0, 7000, new=33, width=512),
        # drafted tokens of a batch, to be verified at once: the cache's bytes count
        _case("chunk_16x4", "chunk", "f16", 32, 8, 128, 16, 500, 2000, new=4),
        # one user's next question behind a short conversation, short heads, odd sizes: latency
        _case("chunk_1x37_d64", "chunk", "bf16", 12, 4, 64, 1, 300, 300, new=37, page=64, group=32),
        # a scheduler's mixed step: a piece of one prompt and the running sequences' next tokens
        _case("chunk_512+31", "chunk", "bf16", 32, 8, 128, 32, 100, 2000, new=1, lead=512, page=32),
        # two chunks of long prompts, wide heads
        _case("chunk_2x700_d256", "chunk", "bf16", 16, 8, 256, 2, 2500, 2500, new=700, group=64),
        # a late chunk of a very long prompt: the matrix unit
        _case("chunk_1x2048_30720", "chunk", "f16", 32, 8, 128, 1, 30720, 30720, new=2048, page=64),
        # a decode step's pages: latency
        _case("summarize_32x1", "summarize", "f16", 32, 8, 128, 32, 512, 640),
        # a long prefill's pages
        _case("summarize_4x2048", "summarize", "f16", 32, 8, 128, 4, 0, 0, new=2048, group=32),
        # a few users with moderate contexts, a quarter of their pages
        _case("sparse_5x4000_d64", "sparse", "bf16", 12, 4, 64, 5, 3000, 4000, group=32, count=64),
        # one very long context on the 70B head layout: 1 / 32 of its pages
        _case("sparse_1x131072", "sparse", "bf16", 64, 8, 128, 1, 131071, 131071, group=64, count=256),
        # a full serving batch with long contexts: 1 / 8 of the pages
        _case("sparse_64x8192", "sparse", "f16", 32, 8, 128, 64, 8191, 8191, count=64),
    ]


def _log(rng, low, high):
    return round(math.exp(rng.uniform(math.log(low), math.log(high))))


def draw(rng):
    kind = rng.choice(("append", "chunk", "chunk", "chunk", "summarize", "sparse", "sparse"))
    while True:
        head = rng.choice((64, 128, 128, 128, 256))
        group = rng.choice([g for g in (32, 64, 128, 256) if g <= head])
        kv_heads = rng.choice((1, 2, 3, 4, 8, 8, 8, 16))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 4, 4, 5, 7, 8, 16))
        dtype = rng.choice(("f16", "bf16"))
        page = rng.choice((16, 16, 32, 64, 128, 256))
        if heads > 128:
            continue
        if kind == "append":
            seqs = _log(rng, 1, 512)
            high = _log(rng, 1, 7000)
            new = rng.choice((0, 1, 1, _log(rng, 1, 300)))
            lead = rng.choice((0, _log(rng, 1, 4000)))
            width = -(-(high + max(new, lead)) // page) + rng.randint(0, 9)
            if lead + (seqs - 1) * new <= 256 * 33 and seqs * width <= 256 * 512:
                return _case(None, kind, dtype, heads, kv_heads, head, seqs, rng.choice((0, high // 2, high)), high, new,
                             lead, page, group, width)
        elif kind == "chunk":
            seqs = _log(rng, 1, 48)
            high = _log(rng, 1, 32768)
            new = rng.choice((1, _log(rng, 2, 16), _log(rng, 2, 2048)))
            lead = rng.choice((0, 0, _log(rng, 1, 2048)))
            most = max(new, lead or new)
            if (lead + (seqs - 1) * new or new) * (high + most) * heads * head <= MOST_SCORES * 128 and \
                    seqs * (high + most) * kv_heads * head <= 1 << 29:
                return _case(None, kind, dtype, heads, kv_heads, head, seqs, rng.choice((0, high // 2, high)), high, new,
                             lead, page, group)
        elif kind == "summarize":
            seqs = _log(rng, 1, 64)
            new = rng.choice((1, _log(rng, 1, 8192)))
            high = _log(rng, 1, 4096)
            if seqs * new * kv_heads * head <= 8192 * 8 * 128 and seqs * high * kv_heads * head <= 1 << 27:
                return _case(None, kind, dtype, heads, kv_heads, head, seqs, rng.choice((0, high)), high, new, 0, page,
                             group)
        else:
            seqs = _log(rng, 1, 64)
            high = _log(rng, 100, 131071)
            count = _log(rng, 2, max(2, high // page))
            if seqs * (high + 1) * kv_heads * _record(head, group) <= 16 * MOST_CACHED and \
                    seqs * heads * min(count * page, high) * head <= 64 * 32 * 1024 * 128:
                return _case(None, kind, dtype, heads, kv_heads, head, seqs, rng.choice((high // 2, high)), high, 1, 0,
                             page, group, count=count)


def _record(head, group):
    return 16 * head + 64 * (head // group + 1)


def _before(case, seed=None):
    """tokens held before the new ones: spread evenly from low to high, in an order that the seed decides"""
    n, low, high = case["seqs"], case["low"], case["high"]
    lens = [high] if n == 1 else [low + (high - low) * i // (n - 1) for i in range(n)]
    if seed is not None:
        random.Random(seed).shuffle(lens)
    return lens


def _new(case):
    return [case["lead"]] + [case["new"]] * (case["seqs"] - 1)


def work(case):
    d, hq, hkv, page, seqs = (case[n] for n in ("head", "heads", "kv_heads", "page", "seqs"))
    before, new = _before(case), _new(case)
    tokens = sum(new)
    kept = hkv * _record(d, case["group"]) / 16  # bytes of one token in the cache
    if case["kind"] == "append":
        # lengths, counts, new lengths, offsets; slots and positions; a page index read and one written per page
        pages = sum(-(-(b + n) // page) - b // page for b, n in zip(before, new))
        return {"bytes": 16 * seqs + 12 * tokens + 8 * pages, "flops": 4 * tokens}
    if case["kind"] == "chunk":
        total = sum(before) + tokens
        pairs = sum(n * b + n * (n + 1) // 2 for b, n in zip(before, new))
        return {"bytes": total * kept + 4 * tokens * hq * d, "flops": 4.0 * pairs * hq * d}
    if case["kind"] == "summarize":
        read = sum((b + n - b // page * page) for b, n in zip(before, new) if n)  # their keys alone
        pages = sum(-(-(b + n) // page) - b // page for b, n in zip(before, new) if n)
        return {"bytes": read * hkv * (d / 2 + 4 * d / case["group"]) + pages * hkv * (d + 4),
                "flops": 3.0 * read * hkv * d}
    pages = [-(-(b + n) // page) for b, n in zip(before, new)]
    scored = sum(n for n in pages if n > case["count"])
    seen = sum(min(b + n, case["count"] * page) for b, n in zip(before, new))
    return {"bytes": scored * hkv * (d + 4) + 4 * sum(pages) + seen * kept + 4 * seqs * hq * d +
            4 * seqs * hkv * case["count"], "flops": 2.0 * scored * hq * d + 4.0 * seen * hq * d}


# ---------------------------------------------------------------- inputs

def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _keys(g, pages, page, kv_heads, d):
    """[pages * page, kv_heads, d]: noise, a few outlier channels, and what a page's tokens have in common"""
    pick = torch.rand((kv_heads, d), generator=g, device="cuda")
    k = _randn(g, pages, page, kv_heads, d) + 0.5 * _randn(g, pages, 1, kv_heads, d)
    k += torch.where(pick < 0.03, torch.where(pick < 0.015, 6.0, -6.0), 0.0)
    return k.flatten(0, 1)


def _filled(case, lens, g, dtype):
    """a cache full of tokens; page table [sequences, longest], every sequence its own pages in random order"""
    page, kv_heads, head = case["page"], case["kv_heads"], case["head"]
    need = [-(-n // page) for n in lens]
    count = sum(need) + 3
    order = torch.randperm(count, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), max(1, max(need))), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    cache = torch.zeros((count, kv_heads, page // 16, _record(head, case["group"])), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (page * kv_heads * head))  # pages filled at a time
    for first in range(0, count, step):
        n = min(count - first, step)
        slots = torch.arange(first * page, (first + n) * page, device="cuda")
        _store(cache, _keys(g, n, page, kv_heads, head).to(dtype), _randn(g, n * page, kv_heads, head).to(dtype), slots)
    return cache, table


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    before, new = _before(case, seed), _new(case)
    lens = [b + n for b, n in zip(before, new)]
    tokens, page = sum(new), case["page"]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    state = {"kind": case["kind"], "page": page, "count": case["count"]}
    if case["kind"] == "append":
        # pages in random order: those that hold the sequences' tokens, and the free ones behind them
        held = [-(-n // page) for n in before]
        needed = sum(-(-n // page) for n in lens) - sum(held)
        order = torch.randperm(sum(held) + needed + 40, generator=g, device="cuda").to(torch.int32)
        table = torch.full((case["seqs"], case["width"]), -1, dtype=torch.int32, device="cuda")
        at = 0
        for i, n in enumerate(held):
            table[i, :n] = order[at:at + n]
            at += n
        # a batch buffer of a captured size, a few rows longer than the batch
        state.update(table=table, lengths=i32(before), counts=i32(new), free=order[at:].contiguous(),
                     free_count=i32([needed + 37]), tokens=tokens + 5)
        return state
    cache, table = _filled(case, lens, g, dtype)
    state.update(cache=cache, table=table, lengths=i32(lens))
    if case["kind"] == "chunk":
        # a slice of the fused projection's output
        heads, kv_heads, head = case["heads"], case["kv_heads"], case["head"]
        x = _randn(g, tokens, (heads + 2 * kv_heads) * head).to(dtype)
        state.update(q=x[:, :heads * head].unflatten(1, (heads, head)), ends=i32([0] + new).cumsum(0).to(torch.int32),
                     lens=lens, new=new)
        return state
    summary = torch.zeros((cache.shape[0], case["kv_heads"], case["head"] + 16), dtype=torch.int8, device="cuda")
    if case["kind"] == "summarize":
        state.update(summary=summary, starts=i32(before), head=case["head"])
        return state
    _summarize(cache, summary, torch.arange(cache.shape[0], device="cuda"), torch.full((cache.shape[0],), page,
                                                                                       device="cuda"))
    state.update(summary=summary, q=_randn(g, case["seqs"], case["heads"], case["head"]).to(dtype))
    return state


# ---------------------------------------------------------------- plain forms

def _shifts(device):
    c = torch.arange(8, device=device, dtype=torch.int32)
    return 4 * (c // 2 + 4 * (c % 2))


def _quantize(x, group):
    """codes int32 [tokens, heads, groups, group]; (scale, minimum) float16 [tokens, heads, groups, 2]"""
    x = x.float().clamp(-LIMIT, LIMIT).unflatten(-1, (-1, group))
    low = x.amin(-1).half()
    scale = ((x.amax(-1) - low.float()) * (1.0 / 15.0)).half()
    s, m = scale.float().unsqueeze(-1), low.float().unsqueeze(-1)
    code = ((x - m) * torch.where(s > 0, 1.0 / s, 0.0)).round().clamp(0.0, 15.0)
    return code.to(torch.int32), torch.stack((scale, low), -1)


def _store(cache, k, v, slots):
    pages, heads, sub, record = cache.shape
    d = k.shape[-1]
    groups = (record - 16 * d) // 64 - 1
    words = cache.view(torch.int32)
    device = cache.device
    at = (slots // (16 * sub)).view(-1, 1, 1), torch.arange(heads, device=device).view(1, -1, 1), (
        slots // 16 % sub).view(-1, 1, 1)
    token = (slots % 16).view(-1, 1, 1)
    kc, kp = _quantize(k, d // groups)
    vc, vp = _quantize(v, d)
    n = torch.arange(d // 8, device=device).view(1, 1, -1)
    shifts = _shifts(device)
    pack = lambda c: (c.reshape(-1, heads, d // 8, 8) << shifts).sum(-1, dtype=torch.int32)  # noqa: E731
    words[(*at, token * (d // 8) + n % 4 * (d // 32) + n // 4)] = pack(kc)
    words[(*at, 2 * d + 16 * torch.arange(groups, device=device).view(1, 1, -1) + token)] = kp.view(torch.int32)[..., 0]
    words[(*at, 2 * d + 16 * groups + 16 * n + token)] = pack(vc)
    words[(*at, 4 * d + 16 * groups + token)] = vp.view(torch.int32)[..., 0]


def _code_keys(records, d):
    """codes, scales and minima of the keys of records [..., record]: [..., 16, groups, d / groups or 1] in 32 bits"""
    groups = (records.shape[-1] - 16 * d) // 64 - 1
    words = records.contiguous().view(torch.int32)
    code = ((words[..., :2 * d].unsqueeze(-1) >> _shifts(records.device)) & 15).float()
    code = code.unflatten(-2, (16, 4, d // 32)).transpose(-2, -3).flatten(-3).unflatten(-1, (groups, -1))
    pair = words[..., 2 * d:2 * d + 16 * groups].contiguous().view(torch.float16).unflatten(-1, (groups, 16, 2))
    pair = pair.transpose(-2, -3).float()
    return code, pair[..., :1], pair[..., 1:]


def _values(records, d):
    """keys and values [..., 16, d] in 32 bits of records [..., record]"""
    code, scale, low = _code_keys(records, d)
    words = records.contiguous().view(torch.int32)[..., -(2 * d + 16):]
    v = ((words[..., :2 * d].unsqueeze(-1) >> _shifts(records.device)) & 15).float()
    v = v.unflatten(-2, (d // 8, 16)).transpose(-2, -3).flatten(-2)
    pair = words[..., 2 * d:].contiguous().view(torch.float16).unflatten(-1, (16, 2)).float()
    return (low + scale * code).flatten(-2), pair[..., 1:] + pair[..., :1] * v


def _softmax(scores, valid):
    scores = scores.masked_fill(~valid, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _append(table, lengths, counts, free, free_count, page, tokens):
    lengths, counts = lengths.long(), counts.long()
    ends = torch.cat((counts.new_zeros(1), counts.cumsum(0))).clamp_max(tokens)
    after = lengths + ends.diff()
    first, last = (lengths + page - 1) // page, (after + page - 1) // page  # new pages' places in the table
    need = last - first
    base = need.cumsum(0) - need
    place = torch.arange(table.shape[1], device=table.device)
    rank = base.view(-1, 1) + place - first.view(-1, 1)
    count = free_count.long()
    taken = torch.where(rank < count, free[(count - 1 - rank).clamp(0, len(free) - 1)], -1)
    fresh = (place >= first.view(-1, 1)) & (place < last.view(-1, 1))
    table.copy_(torch.where(fresh, taken, table))
    row = torch.arange(tokens, device=table.device)
    seq = torch.searchsorted(ends[1:], row, right=True)
    live = seq < len(lengths)
    seq = seq.clamp_max(len(lengths) - 1)
    position = lengths[seq] + row - ends[seq]
    at = table[seq, (position // page).clamp(0, table.shape[1] - 1)].long()
    slots = torch.where(live & (at >= 0), at * page + position % page, -1)
    return (slots, torch.where(live, position, 0).to(torch.int32), ends.to(torch.int32), after.to(torch.int32),
            (count - need.sum()).clamp_min(0).to(torch.int32), table)


def _attend(q, k, v, lengths, rows):
    """q [seqs, rows, heads, d], k and v [seqs, kv_heads, tokens, d]; the last row sees all of a sequence's tokens"""
    b, n, heads, d = q.shape
    kv_heads = k.shape[1]
    qf = q.float().unflatten(2, (kv_heads, -1)).permute(0, 2, 3, 1, 4).reshape(b, kv_heads, -1, d)
    scores = torch.matmul(qf, k.transpose(-1, -2).contiguous()).unflatten(2, (-1, n)) / math.sqrt(d)
    last = (lengths - rows).view(-1, 1, 1, 1, 1) + torch.arange(n, device=q.device).view(-1, 1)
    p = _softmax(scores, torch.arange(k.shape[2], device=q.device) <= last)
    out = torch.matmul(p.flatten(2, 3), v).unflatten(2, (-1, n))
    return out.permute(0, 3, 1, 2, 4).flatten(2, 3).to(q.dtype)


def _tokens(cache, table, d):
    """keys and values [seqs, kv_heads, tokens, d] of the pages table [seqs, width]"""
    k, v = _values(cache[table], d)  # [seqs, pages, kv_heads, sub, 16, d]
    return k.transpose(1, 2).flatten(2, 4), v.transpose(1, 2).flatten(2, 4)


def _chunk(s):
    q, cache, table, page, lens, new = (s[n] for n in ("q", "cache", "table", "page", "lens", "new"))
    d = q.shape[-1]
    if len(set(new)) == 1:  # a batch of equal chunks: padded to its longest sequence
        k, v = _tokens(cache, table, d)
        return _attend(q.unflatten(0, (len(new), -1)), k, v, s["lengths"], new[0]).flatten(0, 1)
    out, at = [], 0
    for i, (n, rows) in enumerate(zip(lens, new)):
        k, v = _tokens(cache, table[i:i + 1, :-(-n // page)], d)
        out.append(_attend(q[at:at + rows].unsqueeze(0), k, v, s["lengths"][i:i + 1], rows)[0])
        at += rows
    return torch.cat(out)


def _summarize(cache, summary, pages, held):
    """the summaries of `pages`, of which `held` tokens count"""
    d, sub = summary.shape[-1] - 16, cache.shape[2]
    step = max(1, (1 << 27) // (16 * sub * cache.shape[1] * d))
    for i in range(0, len(pages), step):
        at = pages[i:i + step]
        code, scale, low = _code_keys(cache[at], d)
        k = (low.double() + scale.double() * code.double()).flatten(-2).flatten(2, 3)  # [pages, kv_heads, page, d]
        valid = torch.arange(16 * sub, device=cache.device) < held[i:i + step].view(-1, 1)
        mean = (k * valid.view(-1, 1, 16 * sub, 1)).sum(2) / held[i:i + step].view(-1, 1, 1)
        codes, unit = _codes(mean)
        summary[at, :, :d] = codes.to(torch.int8)
        summary[at, :, d:d + 4] = unit.float().view(torch.int8)


def _codes(x):
    """whole numbers within +-127 and the power of two [..., 1] that they are multiples of (0 for zeros), in 64 bits"""
    top = x.abs().amax(-1, keepdim=True)
    step = torch.exp2(torch.frexp(top)[1].double() - 7)
    return (x / step).round().clamp(-127, 127), torch.where(top > 0, step, 0.0)


def _touched(table, starts, lengths, page):
    """pages that tokens starts..lengths - 1 went to, and how many tokens of each count"""
    place = torch.arange(table.shape[1], device=table.device)
    s, n = starts.view(-1, 1).long(), lengths.view(-1, 1).long()
    hit = (place >= s // page) & (place < (n + page - 1) // page) & (n > s)
    return table[hit].long(), (n - place * page).clamp_max(page)[hit]


def _select(q, summary, table, lengths, page, count):
    seqs, heads, d = q.shape
    kv_heads, width = summary.shape[1], table.shape[1]
    codes, unit = _codes(q.double().unflatten(1, (kv_heads, -1)))  # [seqs, kv_heads, per, d]
    unit = (unit / unit.amax(2, keepdim=True).clamp_min(1e-300)).clamp_min(2.0 ** -40)
    rec = summary[table]  # [seqs, width, kv_heads, d + 16]
    means = rec[..., :d].float().permute(0, 2, 3, 1).contiguous()
    steps = rec[..., d:d + 4].contiguous().view(torch.float32)[..., 0].permute(0, 2, 1)
    scores = (torch.matmul(codes.float(), means) * unit.float()).amax(2) * steps  # exact
    n = ((lengths.long() + page - 1) // page).view(-1, 1, 1)
    place = torch.arange(width, device=q.device).expand(seqs, kv_heads, width)
    scores = torch.where((place == 0) | (place == n - 1), math.inf, scores).masked_fill(place >= n, -math.inf)
    # ties to the lowest place
    order = torch.sort(scores, dim=-1, descending=True, stable=True)[1][..., :count]
    order = torch.where(order < n, order, width).sort(-1)[0]
    pages = torch.where(order < n, table.unsqueeze(1).expand(-1, kv_heads, -1).gather(2, order.clamp_max(width - 1)), -1)
    if count > width:
        pages = torch.cat((pages, pages.new_full((seqs, kv_heads, count - width), -1)), -1)
    n = n.view(-1)
    return pages, torch.where(n > count, lengths - (n - count) * page, lengths).to(torch.int32)


def _sparse(s):
    q, cache, page = s["q"], s["cache"], s["page"]
    pages, lengths = _select(q, s["summary"], s["table"], s["lengths"], page, s["count"])
    head = torch.arange(cache.shape[1], device=q.device).view(1, -1, 1)
    k, v = _values(cache[pages.clamp_min(0), head], q.shape[-1])  # [seqs, kv_heads, pages, sub, 16, d]
    return pages, lengths, _attend(q.unsqueeze(1), k.flatten(2, 4), v.flatten(2, 4), lengths, 1).squeeze(1)


def _summary_values(s):
    d = s["head"]
    return s["summary"][..., :d] * s["summary"][..., d:d + 4].view(torch.float32)


def run(state):
    s, kind = state, state["kind"]
    if own:
        ga = _attention()
        if kind == "append":
            r = ga.kv4_append(s["table"], s["lengths"], s["counts"], s["free"], s["free_count"], s["page"], s["tokens"])
            return (*r, s["table"])
        if kind == "chunk":
            return ga.kv4_chunk_attention(s["q"], s["cache"], s["table"], s["lengths"], s["ends"])
        if kind == "summarize":
            ga.kv4_summarize(s["cache"], s["summary"], s["table"], s["starts"], s["lengths"])
            return _summary_values(s)
        pages, lengths = ga.kv4_select(s["q"], s["summary"], s["table"], s["lengths"], s["page"], s["count"])
        return pages, lengths, ga.kv4_attention(s["q"], s["cache"], pages, lengths)
    if kind == "append":
        return _append(s["table"], s["lengths"], s["counts"], s["free"], s["free_count"], s["page"], s["tokens"])
    if kind == "chunk":
        return _chunk(s)
    if kind == "summarize":
        _summarize(s["cache"], s["summary"], *_touched(s["table"], s["starts"], s["lengths"], s["page"]))
        return _summary_values(s)
    return _sparse(s)


_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-grinqh-plugin_amd")


def _attention():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import grinqh.attention
    return grinqh.attention


# ---------------------------------------------------------------- definition in 64 bits

def _exact_tokens(cache, pages, head, n, d):
    """the first n tokens' keys and values of one head on the given pages, straight from the bytes"""
    import numpy as np
    rec = cache[pages, head].flatten(0, 1).cpu().numpy()  # [records, record]
    groups = (rec.shape[-1] - 16 * d) // 64 - 1
    nib = np.stack([rec & 15, rec >> 4], -1)  # nibble 2 j and 2 j + 1 of byte j
    c = np.arange(d)
    nibble = c % 8 // 2 + 4 * (c % 2)
    t = np.arange(16)[:, None]
    kbyte = 4 * (t * (d // 8) + c // 8 % 4 * (d // 32) + c // 32) + nibble // 2
    vbyte = 8 * d + 64 * groups + 4 * (c // 8 * 16 + t) + nibble // 2
    pair = lambda at: np.ascontiguousarray(rec[..., at:at + 64]).view(np.float16).astype(np.float64)  # noqa: E731
    kp = np.stack([pair(8 * d + 64 * j) for j in range(groups)], -2)  # [records, groups, 32]
    vp = pair(16 * d + 64 * groups)
    ks, kl = (np.repeat(kp[..., i::2].swapaxes(-1, -2), d // groups, -1) for i in (0, 1))
    k = kl + ks * nib[:, kbyte, nibble % 2]
    v = vp[:, 1::2, None] + vp[:, 0::2, None] * nib[:, vbyte, nibble % 2]
    return tuple(torch.from_numpy(x.reshape(-1, d)[:n]) for x in (k, v))


def _exact_codes(x):
    """8-bit codes along the last axis and their step, numpy float64"""
    import numpy as np
    top = np.abs(x).max(-1, keepdims=True)
    step = np.where(top > 0, 2.0 ** (np.floor(np.log2(np.where(top > 0, top, 1.0))) - 6), 0.0)
    # log2 next to a power of two may round across it
    step = np.where(top >= step * 128, step * 2, np.where((top > 0) & (top < step * 64), step / 2, step))
    return np.clip(np.rint(x / np.where(step > 0, step, 1.0)), -127, 127), step


def _exact_select(q, summary, table, n, count):
    """places of the selected pages of one sequence and head: q numpy [per, d], n pages"""
    import numpy as np
    if n <= count:
        return list(range(n))
    d = q.shape[-1]
    codes, steps = _exact_codes(q)
    steps = np.maximum(steps / max(steps.max(), 1e-300), 2.0 ** -40)
    rec = summary[table[:n]]
    unit = np.ascontiguousarray(rec[:, d:d + 4]).view(np.float32)[:, 0].astype(np.float64)
    score = ((codes @ rec[:, :d].T.astype(np.float64)) * steps).max(0) * unit
    middle = sorted(range(1, n - 1), key=lambda i: (-score[i], i))[:count - 2]
    return [0] + sorted(middle) + [n - 1]


def exact(case, seed):
    import numpy as np
    s = prepare(case, seed)
    page, d, hkv = case["page"], case["head"], case["kv_heads"]
    per = case["heads"] // hkv
    if case["kind"] == "append":
        table, before, new = s["table"].tolist(), s["lengths"].tolist(), s["counts"].tolist()
        free = s["free"].tolist()[:int(s["free_count"])]
        slots, positions, ends, after = [], [], [0], []
        for row, b, n in zip(table, before, new):
            for i in range(b, b + n):
                if i % page == 0:
                    row[i // page] = free.pop()
                slots.append(row[i // page] * page + i % page)
                positions.append(i)
            ends.append(ends[-1] + n)
            after.append(b + n)
        pad = s["tokens"] - len(slots)
        ints = lambda x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
        return (torch.tensor(slots + [-1] * pad), ints(positions + [0] * pad), ints(ends), ints(after),
                ints([len(free)]), ints(table))
    lens, cache = s["lengths"].tolist(), s["cache"]
    if case["kind"] == "chunk":
        if sum(lens) * hkv * d > 1 << 26:
            return None
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        at = 0
        for i, (n, rows) in enumerate(zip(lens, s["new"])):
            pages = s["table"][i, :-(-n // page)].long()
            hide = torch.arange(n, device="cuda") > torch.arange(n - rows, n, device="cuda").view(-1, 1)
            for h in range(hkv if rows else 0):
                k, v = (x.cuda() for x in _exact_tokens(cache, pages, h, n, d))
                for j in range(h * per, (h + 1) * per):
                    z = (s["q"][at:at + rows, j].double() @ k.T) * d ** -0.5
                    out[at:at + rows, j] = torch.softmax(z.masked_fill(hide, -torch.inf), -1) @ v
            at += rows
        return out
    if case["kind"] == "summarize":
        out = np.zeros((cache.shape[0], hkv, d))
        for i, (b, n) in enumerate(zip(s["starts"].tolist(), lens)):
            for j in range(b // page, -(-n // page) if n > b else 0):
                at = int(s["table"][i, j])
                for h in range(hkv):
                    k, _ = _exact_tokens(cache, torch.tensor([at]).cuda(), h, min(page, n - j * page), d)
                    codes, step = _exact_codes(k.numpy().sum(0) / len(k))
                    out[at, h] = codes * step
        return torch.from_numpy(out)
    summary, table = s["summary"].cpu().numpy(), s["table"].cpu().numpy()
    pages = torch.full((case["seqs"], hkv, case["count"]), -1, dtype=torch.int32)
    out = torch.zeros(s["q"].shape, dtype=torch.float64)
    lengths = []
    for i, n in enumerate(lens):
        held = -(-n // page)
        seen = n - max(held - case["count"], 0) * page
        lengths.append(seen)
        for h in range(hkv):
            q = s["q"][i, h * per:(h + 1) * per].double().cpu()
            places = _exact_select(q.numpy(), summary[:, h], table[i], held, case["count"])
            pages[i, h, :len(places)] = torch.from_numpy(table[i][places])
            k, v = _exact_tokens(cache, pages[i, h, :len(places)].long().cuda(), h, seen, d)
            out[i, h * per:(h + 1) * per] = torch.softmax(q @ k.T * d ** -0.5, -1) @ v
    return pages, torch.tensor(lengths, dtype=torch.int32), out
