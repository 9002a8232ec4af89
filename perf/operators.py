"""The attention that belongs between a model's quantized linears, as it is timed: a key/value cache held in 4 bits
(filled, read back, attended to one token per sequence) and the attention over whole prompts.

A case is a dict of plain values.  ``kind`` says what one pass runs:

* ``store``: ``kv4_store`` of new tokens' keys and values at their slots, then ``kv4_load`` of the same slots (what a
  later prompt that shares the prefix does).  A share of the slots is -1 (padding): skipped, and read as zeros.
* ``decode``: ``kv4_attention``, one query token per sequence over its pages.
* ``prompt``: ``prompt_attention`` over packed sequences, causal, query rows aligned with the end of their keys
  (``prefix``: keys that were cached before the prompt's own).

The cache is uint8 [pages, key/value heads, page / 16, record]; a record holds 16 tokens of one head, D channels in
G = D / group groups for the keys and one group for the values:

    keys     16 tokens x D / 8 words; word (channel / 8) % 4 * (D / 32) + channel / 32 of a token
    (scale, minimum) of the keys     G x 16 tokens, float16 pairs
    values   D / 8 words x 16 tokens; word channel / 8
    (scale, minimum) of the values   16 tokens, float16 pairs

Channel c of a word's 8 is its nibble c / 2 + 4 * (c % 2).  With all values limited to +-65504, in 32 bits:
minimum = f16(min), scale = f16((max - minimum) * (1 / 15)), code = round((x - minimum) * (1 / scale)) within 0..15
(0 where the scale is 0), and what a code stands for is minimum + scale * code.  A group that holds a NaN is NaN.

Head counts, head sizes and lengths are those of bench.py's models (Llama-3-8B: 32 query and 8 key/value heads of 128
channels, Llama-3-70B: 64 and 8; prompts of 512 tokens at batch 32, prefills of up to 8192 rows) and generic ones.
Queries, keys and values are slices of one fused projection, as qkv_proj leaves them: N(0, 1), keys with a per-channel
offset of +-6 in 3 % of their channels.
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
# a decode batch's bytes and a prompt's score matrix: the largest listed cases
MOST_DECODE = 64 * 8192 * 8 * 2176
MOST_SCORES = 32 * 8192 * 8192


def _case(name, kind, dtype, heads, kv_heads, head, seqs, low, high, page=16, group=0, prefix=0, skip=0.0):
    """low..high: tokens of the shortest and the longest sequence (store: new tokens in all)"""
    c = {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "head": head, "seqs": seqs, "low": low,
         "high": high, "page": page, "group": group or head, "prefix": prefix, "skip": skip}
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one decode step's new tokens, one per sequence of a batch: latency
        _case("store_32tokens", "store", "f16", 32, 8, 128, 32, 1, 1),
        # odd count, short heads, padded rows of a captured batch size
        _case("store_777tokens_d64", "store", "bf16", 12, 4, 64, 1, 777, 777, page=64, group=32, skip=0.1),
        # a long prefill written at once
        _case("store_8192tokens", "store", "bf16", 32, 8, 128, 4, 2048, 2048, group=32),
        # one user at the start of a chat: latency
        _case("decode_1x500", "decode", "f16", 32, 8, 128, 1, 500, 500),
        # the benchmark's decode batch: 512-token prompts and what they have generated so far
        _case("decode_32x512", "decode", "bf16", 32, 8, 128, 32, 512, 640),
        # a batch of many short and some empty sequences, one head per key/value head, short heads
        _case("decode_100x300_d64", "decode", "f16", 8, 8, 64, 100, 0, 300, page=64, group=32),
        # one very long context on the 70B head layout: work split over the length
        _case("decode_1x131072", "decode", "bf16", 64, 8, 128, 1, 131072, 131072, page=64, group=64),
        # a full serving batch with long contexts: bandwidth
        _case("decode_64x8192", "decode", "f16", 32, 8, 128, 64, 8192, 8192, page=32),
        # a one-line question: latency
        _case("prompt_1x33", "prompt", "f16", 32, 8, 128, 1, 33, 33),
        # a packed batch of prompts of different lengths
        _case("prompt_8x512", "prompt", "f16", 32, 8, 128, 8, 100, 900),
        # a chunk of a long prompt whose first part is cached, wide heads
        _case("prompt_2x700_d256", "prompt", "bf16", 16, 8, 256, 2, 700, 700, prefix=2500),
        # one long prompt
        _case("prompt_1x8192", "prompt", "bf16", 32, 8, 128, 1, 8192, 8192),
    ]


def draw(rng):
    kind = rng.choice(("store", "decode", "decode", "prompt", "prompt"))
    while True:
        head = rng.choice((64, 128, 128, 128, 256))
        group = rng.choice([g for g in (32, 64, 128, 256) if g <= head])
        kv_heads = rng.choice((1, 2, 3, 4, 8, 8, 8, 16))
        heads = kv_heads * rng.choice((1, 2, 3, 4, 4, 4, 5, 7, 8, 16))
        if 3072 in (heads * head, (heads + 2 * kv_heads) * head):
            continue  # row lengths of the projection
        dtype = rng.choice(("f16", "bf16"))
        page = rng.choice((16, 16, 32, 64, 128, 256))
        if kind == "store":
            high = round(math.exp(rng.uniform(0.0, math.log(8192.0))))
            if heads <= 128 and high * kv_heads * head <= 8192 * 8 * 128:
                return _case(None, kind, dtype, heads, kv_heads, head, 1, high, high, page, group,
                             skip=rng.choice((0.0, 0.0, 0.2)))
        elif kind == "decode":
            seqs = round(math.exp(rng.uniform(0.0, math.log(128.0))))
            high = round(math.exp(rng.uniform(0.0, math.log(131072.0))))
            low = rng.choice((0, high // 2, high))
            if (seqs * high * kv_heads * _record(head, group) / 16 <= MOST_DECODE
                    and seqs * heads * high <= 64 * 32 * 8192 and heads <= 128):
                return _case(None, kind, dtype, heads, kv_heads, head, seqs, low, high, page, group)
        else:
            seqs = round(math.exp(rng.uniform(0.0, math.log(32.0))))
            high = round(math.exp(rng.uniform(0.0, math.log(8192.0))))
            low = rng.choice((0, high // 3, high))
            prefix = rng.choice((0, 0, 0, rng.randint(1, 4096)))
            total = sum(_lengths(seqs, low, high))
            if total and total * (total + seqs * prefix) * heads * head <= MOST_SCORES * 128 and heads <= 64:
                return _case(None, kind, dtype, heads, kv_heads, head, seqs, low, high, prefix=prefix)


def _record(head, group):
    return 16 * head + 64 * (head // group + 1)


def _lengths(seqs, low, high):
    """lengths spread evenly from low to high, the ends included"""
    if seqs == 1:
        return [high]
    return [low + (high - low) * i // (seqs - 1) for i in range(seqs)]


def _ragged(case, seed):
    """the case's lengths in an order that the seed decides"""
    lens = _lengths(case["seqs"], case["low"], case["high"])
    random.Random(seed).shuffle(lens)
    return lens


def work(case):
    d, hq, hkv = case["head"], case["heads"], case["kv_heads"]
    lens = _lengths(case["seqs"], case["low"], case["high"])
    total = sum(lens)
    row = d * 2
    kept = hkv * _record(d, case["group"]) / 16  # bytes of one token in the cache
    if case["kind"] == "store":
        # read k and v, write their codes, read them, write k and v; about 8 operations per value each way
        return {"bytes": total * (8 + 4 * hkv * row + 2 * kept), "flops": total * 2 * hkv * d * 16}
    if case["kind"] == "decode":
        return {"bytes": total * kept + 2 * case["seqs"] * hq * row, "flops": 4.0 * total * hq * d}
    p = case["prefix"]
    pairs = sum(n * (n + 1) // 2 + n * p for n in lens)
    return {"bytes": total * 2 * hq * row + 2 * (total + len(lens) * p) * hkv * row, "flops": 4.0 * pairs * hq * d}


# ---------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _projection(g, tokens, heads, kv_heads, head, dtype):
    """q, k, v of a fused projection's output: slices, token rows (heads + 2 kv_heads) * head apart"""
    x = torch.randn((tokens, (heads + 2 * kv_heads) * head), generator=g, device="cuda")
    q, k, v = x.split((heads * head, kv_heads * head, kv_heads * head), 1)
    pick = torch.rand((kv_heads * head,), generator=g, device="cuda")
    k += torch.where(pick < 0.03, torch.where(pick < 0.015, 6.0, -6.0), 0.0)
    q, k, v = x.to(dtype).split((heads * head, kv_heads * head, kv_heads * head), 1)
    return q.unflatten(1, (heads, head)), k.unflatten(1, (kv_heads, head)), v.unflatten(1, (kv_heads, head))


def _pages(case, lens, g):
    """page table [sequences, longest], every sequence its own pages in random order; and the number of pages"""
    page = case["page"]
    need = [-(-n // page) for n in lens]
    count = sum(need) + 3
    order = torch.randperm(count, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros((len(lens), max(1, max(need))), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, count


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    heads, kv_heads, head, page, group = (case[n] for n in ("heads", "kv_heads", "head", "page", "group"))
    lens = _ragged(case, seed)
    state = {"kind": case["kind"], "dtype": dtype}
    if case["kind"] == "prompt":
        before = [case["prefix"] if n else 0 for n in lens]
        q, k, v = _projection(g, sum(lens), heads, kv_heads, head, dtype)
        if any(before):  # keys and values that were cached come as tensors of their own
            _, k, v = _projection(g, sum(lens) + sum(before), 0, kv_heads, head, dtype)
        ends = torch.tensor([[0] + lens, [0] + [n + p for n, p in zip(lens, before)]], device="cuda")
        ends = ends.cumsum(1).to(torch.int32)
        state.update(q=q, k=k, v=v, ends=ends[0].contiguous(), key_ends=ends[1].contiguous())
        return state
    record = _record(head, group)
    if case["kind"] == "store":
        table, count = _pages(case, lens, g)
        cache = torch.zeros((count, kv_heads, page // 16, record), dtype=torch.uint8, device="cuda")
        at = torch.cat([torch.arange(n) for n in lens]).cuda()
        if case["high"] == 1:  # a decode step: each new token stands somewhere in its sequence's last page
            at = torch.randint(0, page, (len(lens),), generator=g, device="cuda")
            slots = table[:, 0] * page + at
        else:
            row = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)]).cuda()
            slots = table[row, at // page] * page + at % page
        slots = slots.to(torch.int64)
        if case["skip"]:
            slots[torch.rand(slots.shape, generator=g, device="cuda") < case["skip"]] = -1
        _, k, v = _projection(g, len(slots), heads, kv_heads, head, dtype)
        state.update(cache=cache, k=k, v=v, slots=slots)
        return state
    table, count = _pages(case, lens, g)
    cache = torch.zeros((count, kv_heads, page // 16, record), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (page * kv_heads * head))  # pages filled at a time
    for first in range(0, count, step):
        slots = torch.arange(first * page, min(count, first + step) * page, device="cuda")
        _, k, v = _projection(g, len(slots), 0, kv_heads, head, dtype)
        _store(cache, k, v, slots)
    q, _, _ = _projection(g, len(lens), heads, kv_heads, head, dtype)
    state.update(cache=cache, q=q, table=table, lengths=torch.tensor(lens, dtype=torch.int32, device="cuda"))
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
    return code.nan_to_num(0.0).to(torch.int32), torch.stack((scale, low), -1)


def _store(cache, k, v, slots):
    pages, heads, sub, record = cache.shape
    d = k.shape[-1]
    groups = (record - 16 * d) // 64 - 1
    keep = slots >= 0
    k, v, slots = k[keep], v[keep], slots[keep]
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


def _values(records, d):
    """keys and values [..., 16, d] in 32 bits of records [..., record]"""
    groups = (records.shape[-1] - 16 * d) // 64 - 1
    words = records.contiguous().view(torch.int32)
    kw, kp, vw, vp = words.split((2 * d, 16 * groups, 2 * d, 16), -1)
    shifts = _shifts(records.device)
    code = lambda w: ((w.unsqueeze(-1) >> shifts) & 15).float()  # noqa: E731
    k = code(kw.unflatten(-1, (16, 4, d // 32))).transpose(-2, -3).flatten(-3)  # [..., 16, d]
    kp = kp.contiguous().view(torch.float16).unflatten(-1, (groups, 16, 2)).transpose(-2, -3).float()
    k = kp[..., 1:] + kp[..., :1] * k.unflatten(-1, (groups, -1))
    v = code(vw.unflatten(-1, (d // 8, 16)).transpose(-1, -2)).flatten(-2)
    vp = vp.contiguous().view(torch.float16).unflatten(-1, (16, 2)).float()
    return k.flatten(-2), vp[..., 1:] + vp[..., :1] * v


def _load(cache, slots, d, dtype):
    pages, heads, sub, record = cache.shape
    at = slots.clamp_min(0)
    records = cache[at // (16 * sub), :, at // 16 % sub]  # [tokens, heads, record]
    k, v = _values(records, d)
    token = (at % 16).view(-1, 1, 1, 1).expand(-1, heads, 1, d)
    keep = (slots >= 0).view(-1, 1, 1)
    return tuple(torch.where(keep, x.gather(2, token).squeeze(2), 0.0).to(dtype) for x in (k, v))


def _softmax(scores, valid):
    scores = scores.masked_fill(~valid, -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-30)


def _decode(q, cache, table, lengths):
    b, heads, d = q.shape
    kv_heads = cache.shape[1]
    k, v = _values(cache[table], d)  # [b, pages, kv_heads, sub, 16, d]
    k = k.transpose(1, 2).flatten(2, 4)
    v = v.transpose(1, 2).flatten(2, 4)  # [b, kv_heads, tokens, d]
    scores = torch.matmul(q.float().view(b, kv_heads, -1, d), k.transpose(-1, -2)) / math.sqrt(d)
    valid = torch.arange(k.shape[2], device=q.device) < lengths.view(-1, 1, 1, 1)
    return torch.matmul(_softmax(scores, valid), v).flatten(1, 2).to(q.dtype)


def _prompt(q, k, v, ends, key_ends):
    tokens, heads, d = q.shape
    keys, kv_heads, _ = k.shape
    row, key = torch.arange(tokens, device=q.device), torch.arange(keys, device=q.device)
    row_seq = torch.searchsorted(ends, row.to(torch.int32), right=True).view(-1, 1)
    key_seq = torch.searchsorted(key_ends, key.to(torch.int32), right=True).view(1, -1)
    # distance from the end of the sequence: a row sees the keys that are at least as far
    valid = (row_seq == key_seq) & (key_ends[key_seq] - key >= ends[row_seq] - row.view(-1, 1))
    qf = q.float().transpose(0, 1).reshape(kv_heads, -1, d)
    scores = torch.matmul(qf, k.float().permute(1, 2, 0)).view(heads, tokens, keys) / math.sqrt(d)
    p = _softmax(scores, valid).view(kv_heads, -1, keys)
    return torch.matmul(p, v.float().transpose(0, 1)).view(heads, tokens, d).transpose(0, 1).to(q.dtype)


def run(state):
    kind = state["kind"]
    if own:
        ga = _attention()
        if kind == "store":
            ga.kv4_store(state["cache"], state["k"], state["v"], state["slots"])
            return ga.kv4_load(state["cache"], state["slots"], state["dtype"])
        if kind == "decode":
            return ga.kv4_attention(state["q"], state["cache"], state["table"], state["lengths"])
        return ga.prompt_attention(state["q"], state["k"], state["v"], state["ends"], state["key_ends"])
    if kind == "store":
        _store(state["cache"], state["k"], state["v"], state["slots"])
        return _load(state["cache"], state["slots"], state["k"].shape[-1], state["dtype"])
    if kind == "decode":
        return _decode(state["q"], state["cache"], state["table"], state["lengths"])
    return _prompt(state["q"], state["k"], state["v"], state["ends"], state["key_ends"])


_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-grinqh-plugin_amd")


def _attention():
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import grinqh.attention
    return grinqh.attention


# ---------------------------------------------------------------- definition in 64 bits

def _exact_codec(x, group):
    """what the codes of x [tokens, heads, d] stand for"""
    t, h, d = x.shape
    x = torch.clip(x.double(), -LIMIT, LIMIT).reshape(t, h, d // group, group)
    low = x.min(-1, keepdim=True).values.to(torch.float16).double()
    step = ((x.max(-1, keepdim=True).values - low) / 15.0).to(torch.float16).double()
    code = torch.where(step > 0, torch.round((x - low) / torch.where(step > 0, step, 1.0)), 0.0)
    return (low + step * torch.clip(code, 0, 15)).reshape(t, h, d)


def _exact_head(q, k, v, first):
    """softmax(q k^T / sqrt(d)) v of one sequence and one key/value head; row i sees keys 0 .. first + i"""
    n = torch.arange(q.shape[-2], device=q.device).view(-1, 1) + first
    s = (q @ k.T) * q.shape[-1] ** -0.5
    s = torch.where(torch.arange(k.shape[0], device=q.device) <= n, s, -torch.inf)
    return torch.softmax(s, -1) @ v


def _exact_token(cache, page, head, sub, d):
    """the 16 tokens of one record of every page of one sequence, straight from the bytes"""
    rec = cache[page, head, sub].cpu().numpy()
    groups = (rec.shape[-1] - 16 * d) // 64 - 1
    import numpy as np
    nib = np.stack([rec & 15, rec >> 4], -1)  # nibble 2 j and 2 j + 1 of byte j
    c = np.arange(d)
    nibble = c % 8 // 2 + 4 * (c % 2)
    t = np.arange(16)[:, None]
    kbyte = 4 * (t * (d // 8) + c // 8 % 4 * (d // 32) + c // 32) + nibble // 2
    vbyte = 8 * d + 64 * groups + 4 * (c // 8 * 16 + t) + nibble // 2
    pair = lambda at: np.ascontiguousarray(rec[..., at:at + 64]).view(np.float16).astype(np.float64)  # noqa: E731
    kp = np.stack([pair(8 * d + 64 * j) for j in range(groups)], -2)  # [pages, groups, 32]
    vp = pair(16 * d + 64 * groups)
    ks, kl = (np.repeat(kp[..., i::2].swapaxes(-1, -2), d // groups, -1) for i in (0, 1))
    k = kl + ks * nib[:, kbyte, nibble % 2]
    v = vp[:, 1::2, None] + vp[:, 0::2, None] * nib[:, vbyte, nibble % 2]
    return torch.from_numpy(k), torch.from_numpy(v)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "store":
        keep = (s["slots"] >= 0).view(-1, 1, 1)
        return tuple(torch.where(keep, _exact_codec(x, g), 0.0)
                     for x, g in ((s["k"], case["group"]), (s["v"], case["head"])))
    hkv, d = case["kv_heads"], case["head"]
    per = case["heads"] // hkv
    if case["kind"] == "decode":
        page = case["page"]
        if sum(_lengths(case["seqs"], case["low"], case["high"])) * hkv * d > 1 << 27:
            return None
        out = torch.zeros((case["seqs"], case["heads"], d), dtype=torch.float64)
        for i, n in enumerate(s["lengths"].tolist()):
            table = s["table"][i, :-(-n // page)].long()
            for h in range(hkv if n else 0):
                parts = [_exact_token(s["cache"], table, h, j, d) for j in range(page // 16)]
                k, v = (torch.stack([x[j] for x in parts], 1).reshape(-1, d)[:n].cuda() for j in (0, 1))
                q = s["q"][i, h * per:(h + 1) * per].double()
                out[i, h * per:(h + 1) * per] = (torch.softmax(q @ k.T * d ** -0.5, -1) @ v).cpu()
        return out
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    a, b = s["ends"].tolist(), s["key_ends"].tolist()
    for i in range(case["seqs"]):
        first = (b[i + 1] - b[i]) - (a[i + 1] - a[i])
        for h in range(case["heads"] if a[i + 1] > a[i] else 0):
            k, v = (s[x][b[i]:b[i + 1], h // per].double() for x in ("k", "v"))
            out[a[i]:a[i + 1], h] = _exact_head(s["q"][a[i]:a[i + 1], h].double(), k, v, first)
    return out
