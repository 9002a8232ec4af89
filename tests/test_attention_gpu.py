"""GPU tests of the attention operators (csrc/kv4.hip, csrc/prompt.hip,
grinqh/attention.py) against plain implementations in 64 bits.

Storing is exact: the cache's bytes equal those of the layout's definition
computed in fp32 with numpy.  The attentions are held to worst-case bounds of
their arithmetic: the weights' rounding to 16 bits (unit roundoff u of their
type) times the sum of the magnitudes they multiply, the logits' fp32 error
(2^-20 of the magnitudes a logit sums, four times the roundoff of a sum of
some ten partial sums) carried through the exponential, and one rounding of
the result."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f16": torch.float16, "bf16": torch.bfloat16}
U = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8}
LIMIT = 65504.0


@pytest.fixture(scope="module", autouse=True)
def _gpu():
    if not torch.cuda.is_available():
        pytest.fail("GPU tests need a HIP device")


def _randn(rng, *shape, dtype="f16", scale=1.0):
    return (torch.from_numpy(rng.standard_normal(shape).astype(np.float32)) * scale).to(DT[dtype]).cuda()


# ---------------------------------------------------------------- the codec in fp32 (numpy)

def _quantize(x, group):
    """codes uint32 [T, H, D], scale and minimum fp16 [T, H, G] of fp32 x"""
    t, h, d = x.shape
    nan = np.isnan(x).reshape(t, h, d // group, group).any(-1)
    x = np.clip(np.nan_to_num(x, nan=0.0, posinf=LIMIT, neginf=-LIMIT), -LIMIT, LIMIT).astype(np.float32)
    g = x.reshape(t, h, d // group, group)
    low = (g.min(-1) + np.float32(0.0)).astype(np.float16)  # a zero is kept as +0
    m = low.astype(np.float32)
    scale = ((g.max(-1) - m) * np.float32(1.0 / 15.0) + np.float32(0.0)).astype(np.float16)
    s = scale.astype(np.float32)
    inv = np.where(s > 0, np.float32(1.0) / np.where(s > 0, s, np.float32(1.0)), np.float32(0.0)).astype(np.float32)
    code = np.clip(np.rint((g - m[..., None]) * inv[..., None]), 0, 15).astype(np.uint32)
    code[nan] = 0
    scale[nan] = np.uint16(0x7E00).view(np.float16)
    low[nan] = np.uint16(0x7E00).view(np.float16)
    return code.reshape(t, h, d), scale, low


def _words(code):
    """8 channels' codes as the word they are kept in: channel c is nibble c / 2 + 4 (c % 2)"""
    t, h, d = code.shape
    c = np.arange(8)
    return (code.reshape(t, h, d // 8, 8) << (4 * (c // 2 + 4 * (c % 2))).astype(np.uint32)).sum(-1, dtype=np.uint32)


def _store_ref(cache, k, v, slots, group):
    """cache: numpy uint8 [pages, heads, sub, record], written in place"""
    pages, heads, sub, record = cache.shape
    d = k.shape[-1]
    groups = d // group
    w = cache.view(np.uint32)
    kc, ks, kl = _quantize(k, group)
    vc, vs, vl = _quantize(v, d)
    kw, vw = _words(kc), _words(vc)
    pair = lambda s, l: s.view(np.uint16).astype(np.uint32) | (l.view(np.uint16).astype(np.uint32) << 16)
    kp, vp = pair(ks, kl), pair(vs, vl)
    n = np.arange(d // 8)
    for t, slot in enumerate(slots):
        if not 0 <= slot < pages * sub * 16:
            continue
        rec = w[slot // (16 * sub), :, slot // 16 % sub]
        tok = int(slot % 16)
        rec[:, tok * (d // 8) + n % 4 * (d // 32) + n // 4] = kw[t]
        rec[:, 2 * d + 16 * np.arange(groups) + tok] = kp[t]
        rec[:, 2 * d + 16 * groups + 16 * n + tok] = vw[t]
        rec[:, 4 * d + 16 * groups + tok] = vp[t][:, 0]


def _params(x, group):
    """(scale * code, minimum) of what is kept of x, fp64 [T, H, D]"""
    t, h, d = x.shape
    c, s, m = _quantize(x, group)
    wide = lambda a: np.repeat(a.astype(np.float64), group, -1)
    return wide(s) * c, wide(m)


LAYOUTS = [("f16", 128, 128, 16, 8), ("bf16", 128, 32, 32, 2), ("f16", 64, 32, 64, 3), ("bf16", 64, 64, 16, 1),
           ("f16", 256, 256, 16, 2), ("bf16", 256, 32, 256, 1), ("f16", 128, 64, 128, 5), ("bf16", 256, 64, 16, 1),
           ("f16", 256, 128, 32, 1)]


def _kv(rng, tokens, heads, kv_heads, d, dtype, aligned=True):
    """k, v as slices of a fused projection (aligned) or of odd rows"""
    pad = 0 if aligned else 1
    x = _randn(rng, tokens, (heads + 2 * kv_heads) * d + pad, dtype=dtype)
    return (x[:, (heads + i * kv_heads) * d:][:, :kv_heads * d].unflatten(1, (kv_heads, d)) for i in (0, 1))


@pytest.mark.parametrize("dtype,d,group,page,heads", LAYOUTS)
@pytest.mark.parametrize("tokens", [1, 37])
def test_store_and_load(dtype, d, group, page, heads, tokens):
    from grinqh import attention as ga
    rng = np.random.default_rng(d + group + tokens)
    pages = max(3, 80 // page)
    cache = ga.kv4_cache(pages, heads, d, page, group)
    before = rng.integers(0, 256, cache.shape, dtype=np.uint8)
    cache.copy_(torch.from_numpy(before))
    k, v = _kv(rng, tokens, heads + 1, heads, d, dtype, aligned=tokens > 1)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    if tokens > 4:
        slots[3], slots[7], slots[11] = -1, pages * page, 1 << 40  # padding, and behind the cache
    st = torch.from_numpy(slots).cuda()
    ga.kv4_store(cache, k, v, st)
    kf, vf = k.float().cpu().numpy(), v.float().cpu().numpy()
    _store_ref(before, kf, vf, slots, group)
    assert np.array_equal(cache.cpu().numpy(), before)
    for out_dtype in DT.values():
        k2, v2 = ga.kv4_load(cache, st, out_dtype)
        keep = ((slots >= 0) & (slots < pages * page))[:, None, None]
        for got, x, g in ((k2, kf, group), (v2, vf, d)):
            sc, m = _params(x, g)
            want = torch.from_numpy(np.where(keep, (m + sc).astype(np.float32), np.float32(0.0))).to(out_dtype)
            assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_store_special_values(dtype):
    """NaN, infinities, constants, values past fp16's range, tiny ones, signed zeros"""
    from grinqh import attention as ga
    rng = np.random.default_rng(3)
    x = rng.standard_normal((12, 1, 128)).astype(np.float32)
    x[0, 0, 5] = np.nan
    x[1, 0, 40] = np.inf
    x[2, 0, 70] = -np.inf
    x[3] = 1.25
    x[4] = 0.0
    x[5] *= 1e-6
    x[6] *= 1e-9 if dtype == "f16" else 1e-30
    x[7] *= 6e4 if dtype == "f16" else 1e30
    x[8, 0, ::2] = -0.0
    x[9, 0, :] = np.where(np.arange(128) % 2, LIMIT, -LIMIT)
    x[10, 0, 3], x[10, 0, 4] = np.nan, np.inf
    x[11] = np.float32(0.5) * np.arange(128)[None] % 16  # ties between codes
    t = torch.from_numpy(x).to(DT[dtype]).cuda()
    cache = ga.kv4_cache(1, 1, 128, 16, 32)
    slots = torch.arange(12).cuda()
    ga.kv4_store(cache, t, t, slots)
    want = np.zeros(cache.shape, np.uint8)
    xf = t.float().cpu().numpy()
    _store_ref(want, xf, xf, np.arange(12), 32)
    assert np.array_equal(cache.cpu().numpy(), want)
    k, v = ga.kv4_load(cache, slots, torch.bfloat16)
    assert bool(k[0, 0, :32].isnan().all()) and not bool(k[0, 0, 32:].isnan().any()) and bool(v[0].isnan().all())
    assert not bool(k[1:10].isnan().any())


def test_cache_past_32_bit_offsets():
    """records, slots and pages more than 2^32 bytes into the cache"""
    from grinqh import attention as ga
    rng = np.random.default_rng(11)
    pages = (5 << 30) // (8 * 2176)
    cache = torch.empty((pages, 8, 1, 2176), dtype=torch.uint8, device="cuda")
    length = 100
    table = torch.tensor([[pages - 1 - i for i in range(7)]], dtype=torch.int32).cuda()
    at = torch.arange(length)
    slots = table[0, at.cuda() // 16].long() * 16 + at.cuda() % 16
    k, v = (_randn(rng, length, 8, 128) for _ in (0, 1))
    ga.kv4_store(cache, k, v, slots)
    k2, v2 = ga.kv4_load(cache, slots)
    sc, m = _params(k.float().cpu().numpy(), 128)
    assert torch.equal(k2.cpu(), torch.from_numpy((sc + m).astype(np.float32)).half())
    q = _randn(rng, 1, 32, 128)
    out = ga.kv4_attention(q, cache, table, torch.tensor([length], dtype=torch.int32).cuda())
    _check_decode(out, q, [(k, v)], 128, "f16")


# ---------------------------------------------------------------- decode

def _check_decode(out, q, seqs, group, dtype, scale=None):
    """out [B, Hq, D] against fp64 from what the cache keeps of each sequence's (k, v) [T, H, D]"""
    out = out.double().cpu().numpy()
    qf = q.double().cpu().numpy()
    b, hq, d = qf.shape
    scale = d ** -0.5 if scale is None else scale
    for i, (k, v) in enumerate(seqs):
        if k.shape[0] == 0:
            assert not out[i].any()
            continue
        t, hkv, _ = k.shape
        per = hq // hkv
        ks, km = _params(k.float().cpu().numpy(), group)
        vs, vm = _params(v.float().cpu().numpy(), d)
        for h in range(hkv):
            qh = qf[i, h * per:(h + 1) * per]
            s = qh @ (ks + km)[:, h].T * scale
            p = np.exp(s - s.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            o = p @ (vs + vm)[:, h]
            size = (np.abs(qh) @ (np.abs(km) + ks)[:, h].T * scale).max(-1, keepdims=True)
            delta = 2.0 ** -20 * (size + 1)
            step = (vs[:, h].max(-1) / 15).max()  # largest value scale (the largest code is 15)
            tol = ((U["f16"] + 2 * delta + 2.0 ** -18) * (p @ (np.abs(vm) + vs)[:, h]) + U[dtype] * np.abs(o)
                   + t * 15 * 2.0 ** -25 * step + 2.0 ** -24)
            err = np.abs(out[i, h * per:(h + 1) * per] - o)
            assert (err <= tol).all(), (i, h, float((err / tol).max()))


def _paged(rng, lens, hkv, d, page, group, dtype, fill=0xFF, scale_v=None, spare=2):
    """A cache whose unwritten bytes are `fill` (0xFF: parameters that are NaN), its table and each sequence's k, v"""
    from grinqh import attention as ga
    need = [-(-n // page) for n in lens]
    pages = sum(need) + spare
    order = rng.permutation(pages).astype(np.int32)
    table = np.full((len(lens), max(1, max(need))), -7, np.int32)  # entries past a sequence's pages are not read
    cache = ga.kv4_cache(pages, hkv, d, page, group)
    cache.fill_(fill)
    seqs, at = [], 0
    for i, n in enumerate(lens):
        table[i, :need[i]] = order[at:at + need[i]]
        at += need[i]
        k, v = (_randn(rng, n, hkv, d, dtype=dtype) for _ in (0, 1))
        k[:, :, ::17] += 6.0
        if scale_v is not None and n:
            v *= torch.from_numpy(scale_v(n)).to(v.dtype).cuda().view(-1, 1, 1)
        seqs.append((k, v))
        if n:
            t = np.arange(n)
            slots = table[i, t // page].astype(np.int64) * page + t % page
            ga.kv4_store(cache, k, v, torch.from_numpy(slots).cuda())
    return cache, torch.from_numpy(table).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), seqs


@pytest.mark.parametrize("dtype,d,group,page,hkv", LAYOUTS)
@pytest.mark.parametrize("per", [1, 4, 7])
def test_decode(dtype, d, group, page, hkv, per):
    from grinqh import attention as ga
    rng = np.random.default_rng(d * 3 + group + per)
    lens = [0, 1, 15, 16, 17, 31, 32, 33, 64, 65, 127, 129, 200, 500]
    cache, table, lengths, seqs = _paged(rng, lens, hkv, d, page, group, dtype)
    q = _randn(rng, len(lens), hkv * per, d, dtype=dtype)
    _check_decode(ga.kv4_attention(q, cache, table, lengths), q, seqs, group, dtype)


@pytest.mark.parametrize("per", [16, 17, 40])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_decode_many_query_heads(per, d):
    from grinqh import attention as ga
    rng = np.random.default_rng(per)
    cache, table, lengths, seqs = _paged(rng, [70, 0, 333], 2, d, 32, 64, "f16")
    q = _randn(rng, 3, 2 * per, d)
    _check_decode(ga.kv4_attention(q, cache, table, lengths), q, seqs, 64, "f16")


@pytest.mark.parametrize("lens", [[2777], [2777, 40, 0], [9000, 1, 513], [0, 0, 5000, 0], [512, 513, 544, 545]])
@pytest.mark.parametrize("hkv,per", [(2, 4), (1, 16), (1, 33), (3, 1)])
def test_decode_split_lengths(lens, hkv, per):
    """few sequences are shared by several blocks; a table with room for more changes nothing but the plan"""
    from grinqh import attention as ga
    rng = np.random.default_rng(17)
    cache, table, lengths, kv = _paged(rng, lens, hkv, 128, 16, 128, "bf16")
    q = _randn(rng, len(lens), hkv * per, 128, dtype="bf16")
    wide = torch.nn.functional.pad(table, (0, 700), value=-1)
    for tab in (table, wide):
        for _ in range(2):  # the counters are zero again after a call
            _check_decode(ga.kv4_attention(q, cache, tab, lengths), q, kv, 128, "bf16")


@pytest.mark.parametrize("seqs", [63, 64, 65, 130, 700, 1024, 1025])
def test_decode_many_sequences(seqs):
    from grinqh import attention as ga
    rng = np.random.default_rng(seqs)
    lens = rng.integers(0, 60, seqs)
    lens[seqs // 3], lens[seqs // 2], lens[-1] = 3000, 0, 700
    cache, table, lengths, kv = _paged(rng, lens.tolist(), 1, 64, 16, 64, "f16")
    q = _randn(rng, seqs, 2, 64)
    _check_decode(ga.kv4_attention(q, cache, table, lengths), q, kv, 64, "f16")


def test_decode_more_units_than_counters():
    """beyond 2^15 (sequence, head) pairs no sequence is shared between blocks"""
    from grinqh import attention as ga
    rng = np.random.default_rng(2)
    cache, table, lengths, kv = _paged(rng, [900, 33], 8, 64, 16, 64, "f16")
    pick = torch.arange(5000).cuda() % 2
    q = _randn(rng, 2, 8, 64)
    out = ga.kv4_attention(q[pick], cache, table[pick], lengths[pick])
    assert torch.equal(out, out[:2][pick])
    _check_decode(out[:2], q, kv, 64, "f16")


@pytest.mark.parametrize("tokens", [48, 4000])
def test_decode_value_scales(tokens):
    """value sizes that differ by 10^7 between tokens, the largest last: the running reference has to follow them;
    tiny ones throughout; constant ones, whose scale is zero"""
    from grinqh import attention as ga
    rng = np.random.default_rng(tokens)
    for sizes in (lambda n: np.geomspace(1e-4, 1e3, n).astype(np.float32),
                  lambda n: np.geomspace(1e3, 1e-4, n).astype(np.float32),
                  lambda n: np.full(n, 2e-5, np.float32), lambda n: np.zeros(n, np.float32)):
        cache, table, lengths, kv = _paged(rng, [tokens], 1, 128, 16, 128, "f16", scale_v=sizes)
        q = _randn(rng, 1, 4, 128)
        _check_decode(ga.kv4_attention(q, cache, table, lengths), q, kv, 128, "f16")


@pytest.mark.parametrize("size", [0.0, 1e-7, 30.0, 1e4])
def test_decode_query_sizes_and_scale(size):
    from grinqh import attention as ga
    rng = np.random.default_rng(5)
    cache, table, lengths, kv = _paged(rng, [90, 1000], 2, 128, 16, 32, "f16")
    q = _randn(rng, 2, 8, 128) * size
    scale = 0.5 / max(1.0, size)
    _check_decode(ga.kv4_attention(q, cache, table, lengths, scale=scale), q, kv, 32, "f16", scale)
    qb = _randn(rng, 2, 8, 128, dtype="bf16") * (size * 1e-25)
    _check_decode(ga.kv4_attention(qb, cache, table, lengths), qb, kv, 32, "bf16")


def test_decode_nan_stays_with_its_head():
    from grinqh import attention as ga
    rng = np.random.default_rng(6)
    cache, table, lengths, kv = _paged(rng, [70, 70], 2, 128, 16, 64, "f16")
    k, v = kv[1]
    k = k.clone()
    k[69, 1, 3] = float("nan")
    t = torch.arange(70).cuda()
    ga.kv4_store(cache, k, v, table[1, t // 16].long() * 16 + t % 16)
    q = _randn(rng, 2, 8, 128)
    out = ga.kv4_attention(q, cache, table, lengths)
    assert bool(out[1, 4:].isnan().all()) and not bool(out[1, :4].isnan().any())
    _check_decode(out[:1], q[:1], kv[:1], 64, "f16")
    q[0, 2, 5] = float("inf")
    out = ga.kv4_attention(q, cache, table, lengths)
    assert not bool(out[0, 2].isfinite().any()) and bool(out[0, :2].isfinite().all())


@pytest.mark.parametrize("length", [40, 5000])
def test_decode_refuses_bad_pages_with_nan(length):
    """a page outside the cache, a length past the table: NaN for that sequence, the others as ever"""
    from grinqh import attention as ga
    rng = np.random.default_rng(7)
    cache, table, lengths, kv = _paged(rng, [length, length], 1, 128, 16, 128, "f16")
    q = _randn(rng, 2, 4, 128)
    for bad in (-1, cache.shape[0], 2 ** 31 - 1, -2 ** 31):
        tab = table.clone()
        tab[1, 1] = bad
        out = ga.kv4_attention(q, cache, tab, lengths)
        assert bool(out[1].isnan().all())
        _check_decode(out[:1], q[:1], kv[:1], 128, "f16")
    longer = lengths.clone()
    longer[1] = table.shape[1] * 16 + 1
    out = ga.kv4_attention(q, cache, table, longer)
    assert bool(out[1].isnan().all())
    _check_decode(out[:1], q[:1], kv[:1], 128, "f16")
    longer[1] = -3
    assert not bool(ga.kv4_attention(q, cache, table, longer)[1].any())


def test_decode_without_pages_or_sequences():
    from grinqh import attention as ga
    empty = ga.kv4_cache(0, 2, 128)
    q = torch.ones((3, 4, 128), dtype=torch.float16, device="cuda")
    table = torch.zeros((3, 2), dtype=torch.int32, device="cuda")
    out = ga.kv4_attention(q, empty, table, torch.tensor([0, 5, 0], dtype=torch.int32).cuda())
    assert not bool(out[0].any()) and bool(out[1].isnan().all()) and not bool(out[2].any())
    none = ga.kv4_attention(q, empty, table[:, :0], torch.zeros(3, dtype=torch.int32).cuda())
    assert not bool(none.any())
    assert ga.kv4_attention(q[:0], empty, table[:0], torch.zeros(0, dtype=torch.int32).cuda()).shape == (0, 4, 128)
    ga.kv4_store(empty, q[:, :2], q[:, :2], torch.zeros(3, dtype=torch.int64).cuda())
    k, v = ga.kv4_load(empty, torch.zeros(3, dtype=torch.int64).cuda())
    assert not bool(k.any()) and not bool(v.any())


def test_decode_strided_queries_and_tables():
    from grinqh import attention as ga
    rng = np.random.default_rng(8)
    cache, table, lengths, kv = _paged(rng, [100, 30], 2, 128, 16, 128, "f16")
    wide = _randn(rng, 2, 3, 10, 128)
    tab = torch.stack((table, table), 2)[:, :, 0]  # columns two apart
    big = torch.full((2, table.shape[1] + 5), -1, dtype=torch.int32).cuda()
    big[:, :table.shape[1]] = table
    for q in (wide[:, 1, 1:9], wide[:, 0, ::2][:, :4], wide.permute(0, 2, 1, 3)[:, :8, 2],
              _randn(rng, 2, 8, 129)[:, :, 1:]):
        for t in (tab, big[:, :table.shape[1]]):
            _check_decode(ga.kv4_attention(q, cache, t, lengths), q, kv, 128, "f16")


# ---------------------------------------------------------------- prompts

def _check_prompt(out, q, k, v, ends, key_ends, dtype, scale=None):
    out = out.double()
    qd, kd, vd = q.double(), k.double(), v.double()
    hq, d = q.shape[1:]
    per = hq // k.shape[1]
    scale = d ** -0.5 if scale is None else scale
    covered = torch.zeros(q.shape[0], dtype=torch.bool, device=q.device)
    for a, b, ka, kb in zip(ends[:-1], ends[1:], key_ends[:-1], key_ends[1:]):
        rows, keys = b - a, kb - ka
        covered[a:b] = True
        if rows == 0:
            continue
        see = torch.arange(keys, device=q.device) <= torch.arange(rows, device=q.device).view(-1, 1) + keys - rows
        for h in range(hq):
            kh, vh = kd[ka:kb, h // per], vd[ka:kb, h // per]
            s = (qd[a:b, h] @ kh.T * scale).masked_fill(~see, -math.inf)
            top = s.amax(-1, keepdim=True) if keys else torch.full((rows, 1), -math.inf, device=q.device)
            p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
            p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
            o = p @ vh
            size = (qd[a:b, h].abs() @ kh.abs().T * scale).amax(-1, keepdim=True) if keys else torch.zeros_like(top)
            delta = 2.0 ** -20 * (size + 1)
            tol = ((U[dtype] + 2 * delta + 2.0 ** -18) * (p @ vh.abs()) + U[dtype] * o.abs()
                   + keys * 2.0 ** -25 * (vh.abs().max() if keys else 0.0) + 2.0 ** -24)
            err = (out[a:b, h] - o).abs()
            assert bool((err <= tol).all()), (a, h, float((err / tol).max()))
    assert not bool(out[~covered].any())


def _ends(lens):
    return [0] + np.cumsum(lens).tolist()


def _dev(ends):
    return torch.tensor(ends, dtype=torch.int32).cuda()


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 2), (6, 3), (16, 1)])
def test_prompt(dtype, d, hq, hkv):
    from grinqh import attention as ga
    rng = np.random.default_rng(d + hq)
    lens = [1, 0, 63, 64, 65, 2, 127, 129, 0, 300]
    ends = _ends(lens)
    x = _randn(rng, ends[-1], (hq + 2 * hkv) * d + 8, dtype=dtype)
    q, k, v = (y.unflatten(1, (-1, d)) for y in x[:, :-8].split((hq * d, hkv * d, hkv * d), 1))
    out = ga.prompt_attention(q, k, v, _dev(ends))
    _check_prompt(out, q, k, v, ends, ends, dtype)


@pytest.mark.parametrize("rows", [1, 31, 32, 33, 128, 255, 256, 257, 600])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_prompt_one_sequence(rows, d):
    from grinqh import attention as ga
    rng = np.random.default_rng(rows)
    q, k, v = _randn(rng, rows, 4, d), _randn(rng, rows, 2, d), _randn(rng, rows, 2, d)
    _check_prompt(ga.prompt_attention(q, k, v, _dev([0, rows])), q, k, v, [0, rows], [0, rows], "f16")


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prompt_with_other_keys(d, dtype):
    """cached keys before the prompt's own; fewer keys than rows (rows that see none); no keys; rows behind the last
    sequence, also where they are all there is"""
    from grinqh import attention as ga
    rng = np.random.default_rng(d)
    rows, keys = [5, 200, 70, 0, 33, 1, 300], [105, 200, 30, 40, 0, 900, 299]
    ends, key_ends = _ends(rows), _ends(keys)
    tail = 77
    q = _randn(rng, ends[-1] + tail, 4, d, dtype=dtype)
    k, v = (_randn(rng, key_ends[-1] + 9, 2, d, dtype=dtype) for _ in (0, 1))
    out = ga.prompt_attention(q, k, v, _dev(ends), _dev(key_ends), scale=0.2)
    _check_prompt(out, q, k, v, ends, key_ends, dtype, 0.2)
    assert not bool(ga.prompt_attention(q, k, v, _dev([0]), _dev([0])).any())
    assert not bool(ga.prompt_attention(q, k[:0], v[:0], _dev([0, 9]), _dev([0, 0])).any())
    assert ga.prompt_attention(q[:0], k, v, _dev([0, 0]), _dev([0, 5])).shape == (0, 4, d)


@pytest.mark.parametrize("seqs", [63, 64, 65, 200])
def test_prompt_many_sequences(seqs):
    from grinqh import attention as ga
    rng = np.random.default_rng(seqs)
    lens = rng.integers(0, 40, seqs)
    lens[seqs // 2] = 400
    ends = _ends(lens)
    q, k, v = _randn(rng, ends[-1], 2, 64), _randn(rng, ends[-1], 1, 64), _randn(rng, ends[-1], 1, 64)
    _check_prompt(ga.prompt_attention(q, k, v, _dev(ends)), q, k, v, ends, ends, "f16")


def test_prompt_nan_and_infinity_stay_with_their_sequence():
    """NaN in other sequences' keys and in keys a row must not see; -inf and +inf logits"""
    from grinqh import attention as ga
    rng = np.random.default_rng(1)
    lens = [100, 90, 30]
    ends = _ends(lens)
    q, k, v = _randn(rng, 220, 8, 128), _randn(rng, 220, 2, 128), _randn(rng, 220, 2, 128)
    clean = ga.prompt_attention(q, k, v, _dev(ends))
    k2, v2 = k.clone(), v.clone()
    k2[100:190], v2[100:190] = float("nan"), float("inf")
    out = ga.prompt_attention(q, k2, v2, _dev(ends))
    assert torch.equal(out[:100], clean[:100]) and torch.equal(out[190:], clean[190:])
    assert bool(out[100:190].isnan().all())
    k3 = k.clone()
    k3[99] = float("nan")  # the last key: its own row alone
    out = ga.prompt_attention(q, k3, v, _dev(ends))
    assert torch.equal(out[:99], clean[:99]) and bool(out[99].isnan().all())
    q4, k4 = q.clone(), k.clone()
    q4[:, :, 0], k4[5, :, 0], k4[:5, :, 0], k4[6:, :, 0] = 1.0, float("-inf"), 0.0, 0.0
    out = ga.prompt_attention(q4, k4, v, _dev(ends))
    v5 = v.clone()
    v5[5] = 1000.0  # a key whose logits are -inf has no weight
    assert bool(out.isfinite().all()) and torch.equal(out[6:], ga.prompt_attention(q4, k4, v5, _dev(ends))[6:])


def test_prompt_large_logits():
    from grinqh import attention as ga
    rng = np.random.default_rng(2)
    q, k, v = _randn(rng, 300, 4, 128, scale=12.0), _randn(rng, 300, 4, 128, scale=12.0), _randn(rng, 300, 4, 128)
    q *= torch.linspace(0.1, 3.0, 300).view(-1, 1, 1).cuda().half()
    k *= torch.linspace(0.1, 3.0, 300).view(-1, 1, 1).cuda().half()  # the reference has to rise over and over
    _check_prompt(ga.prompt_attention(q, k, v, _dev([0, 300])), q, k, v, [0, 300], [0, 300], "f16")


def test_prompt_strides_and_offsets():
    from grinqh import attention as ga
    rng = np.random.default_rng(4)
    x = _randn(rng, 150, 20, 128)
    flipped = _randn(rng, 4, 150, 128).transpose(0, 1)  # heads outermost
    odd = _randn(rng, 150, 4, 129)[:, :, 1:]
    for q, k, v in ((x[:, 0:8], x[:, 8:12], x[:, 12:16]), (x[:, 0:16:2], flipped, x[:, 3:7]),
                    (x[:, 2:10], odd, flipped)):
        _check_prompt(ga.prompt_attention(q, k, v, _dev([0, 90, 150])), q, k, v, [0, 90, 150], [0, 90, 150], "f16")
    for one in (x[:1, 8:12].expand(150, -1, -1), torch.zeros((150, 4, 128), dtype=torch.float16, device="cuda")):
        _check_prompt(ga.prompt_attention(x[:, :8], one, x[:, 8:12], _dev([0, 90, 150])), x[:, :8], one, x[:, 8:12],
                      [0, 90, 150], [0, 90, 150], "f16")
        _check_prompt(ga.prompt_attention(x[:, :8], x[:, 8:12], one, _dev([0, 90, 150])), x[:, :8], x[:, 8:12], one,
                      [0, 90, 150], [0, 90, 150], "f16")
    # offsets past the tensors are limited to them
    q, k, v = x[:, 0:8], x[:, 8:12], x[:, 12:16]
    out = ga.prompt_attention(q, k, v, _dev([-5, 90, 4000]))
    _check_prompt(out, q, k, v, [0, 90, 150], [0, 90, 150], "f16")


def test_prompt_agrees_with_decode():
    """the last row of a prompt over loaded keys and values is what the single-token form gives"""
    from grinqh import attention as ga
    rng = np.random.default_rng(9)
    cache, table, lengths, kv = _paged(rng, [300], 2, 128, 16, 128, "f16")
    t = torch.arange(300).cuda()
    k, v = ga.kv4_load(cache, table[0, t // 16].long() * 16 + t % 16)
    q = _randn(rng, 1, 8, 128)
    a = ga.prompt_attention(q, k, v, _dev([0, 1]), _dev([0, 300])).float()
    b = ga.kv4_attention(q, cache, table, lengths).float()
    assert float((a - b).abs().max()) <= 8 * U["f16"] * float(v.float().abs().max())


# ---------------------------------------------------------------- streams, graphs, repeatability

def test_other_stream_and_repeatable():
    from grinqh import attention as ga
    rng = np.random.default_rng(12)
    cache, table, lengths, kv = _paged(rng, [3000, 10, 700], 2, 128, 16, 128, "f16")
    q, x = _randn(rng, 3, 8, 128), _randn(rng, 500, 12, 128)
    ends = _dev([0, 333, 500])
    first = ga.kv4_attention(q, cache, table, lengths), ga.prompt_attention(x[:, :8], x[:, 8:10], x[:, 10:], ends)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = ga.kv4_attention(q, cache, table, lengths), ga.prompt_attention(x[:, :8], x[:, 8:10], x[:, 10:], ends)
    torch.cuda.current_stream().wait_stream(s)
    for _ in range(3):
        third = ga.kv4_attention(q, cache, table, lengths), ga.prompt_attention(x[:, :8], x[:, 8:10], x[:, 10:], ends)
        for a, b, c in zip(first, again, third):
            assert torch.equal(a, b) and torch.equal(a, c)


def test_graph_replay():
    """a captured decode step: store, attention; replayed with other inputs between eager calls"""
    from grinqh import attention as ga
    rng = np.random.default_rng(13)
    cache, table, lengths, kv = _paged(rng, [2000, 33], 2, 128, 16, 128, "f16", spare=3)
    q, k, v = _randn(rng, 2, 8, 128), _randn(rng, 2, 2, 128), _randn(rng, 2, 2, 128)
    slots = torch.tensor([table[0, 2].item() * 16 + 3, -1]).cuda()
    x = _randn(rng, 200, 12, 128)
    ends = _dev([0, 80, 200])

    def step():
        ga.kv4_store(cache, k, v, slots)
        a = ga.kv4_attention(q, cache, table, lengths)
        return a, ga.prompt_attention(x[:, :8], x[:, 8:10], x[:, 10:], ends), *ga.kv4_load(cache, slots)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        outs = step()
    for i in range(4):
        for t in (q, k, v, x):
            t.copy_(_randn(rng, *t.shape))
        lengths[0] = 2000 - 500 * i
        g.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


# ---------------------------------------------------------------- refusals

def _args():
    from grinqh import attention as ga
    z = lambda *s, dtype=torch.float16: torch.zeros(s, dtype=dtype, device="cuda")
    return ga, ga.kv4_cache(2, 2, 128), z


def test_refusals():
    ga, cache, z = _args()
    i32, i64 = torch.int32, torch.int64
    k, q, slots = z(3, 2, 128), z(3, 8, 128), z(3, dtype=i64)
    table, lengths = z(3, 4, dtype=i32), z(3, dtype=i32)
    bad = [
        lambda: ga.kv4_store(cache.cpu(), k, k, slots),
        lambda: ga.kv4_store(cache, k.cpu(), k, slots),
        lambda: ga.kv4_store(cache, k, k.bfloat16(), slots),
        lambda: ga.kv4_store(cache, k.float(), k.float(), slots),
        lambda: ga.kv4_store(cache, z(3, 4, 128), k, slots),
        lambda: ga.kv4_store(cache, z(3, 2, 64), z(3, 2, 64), slots),
        lambda: ga.kv4_store(cache, k, k[:2], slots),
        lambda: ga.kv4_store(cache, k, k, slots[:2]),
        lambda: ga.kv4_store(cache, k, k, slots.to(i32)),
        lambda: ga.kv4_store(cache[:, :, :, :100], k, k, slots),
        lambda: ga.kv4_store(cache.to(torch.int8), k, k, slots),
        lambda: ga.kv4_store(cache.expand(2, 2, 3, -1), k, k, slots),
        lambda: ga.kv4_store(torch.zeros((2, 2, 3, 2176), dtype=torch.uint8, device="cuda"), k, k, slots),
        lambda: ga.kv4_load(cache, slots, torch.float32),
        lambda: ga.kv4_load(cache, slots.cpu()),
        lambda: ga.kv4_attention(z(3, 7, 128), cache, table, lengths),
        lambda: ga.kv4_attention(z(3, 8, 64), cache, table, lengths),
        lambda: ga.kv4_attention(q[0], cache, table, lengths),
        lambda: ga.kv4_attention(q, cache, table[:2], lengths),
        lambda: ga.kv4_attention(q, cache, table.long(), lengths),
        lambda: ga.kv4_attention(q, cache, table, lengths.long()),
        lambda: ga.kv4_attention(q, cache, table, lengths[:2]),
        lambda: ga.kv4_attention(q, cache, table, lengths, scale=0.0),
        lambda: ga.kv4_attention(q, cache, table, lengths, scale=float("nan")),
        lambda: ga.kv4_attention(q, cache, table, lengths, scale=-1.0),
        lambda: ga.prompt_attention(q, z(3, 3, 128), z(3, 3, 128), lengths),
        lambda: ga.prompt_attention(z(3, 8, 96), z(3, 8, 96), z(3, 8, 96), lengths),
        lambda: ga.prompt_attention(q, k, z(3, 2, 64), lengths),
        lambda: ga.prompt_attention(q, k, k[:2], lengths),
        lambda: ga.prompt_attention(q, z(5, 2, 128), z(5, 2, 128), lengths),
        lambda: ga.prompt_attention(q, k, k, lengths.long()),
        lambda: ga.prompt_attention(q, k, k, lengths[:0]),
        lambda: ga.prompt_attention(q, k, k, lengths, lengths[:2]),
        lambda: ga.prompt_attention(q, k, k, lengths.cpu()),
        lambda: ga.prompt_attention(q, k.bfloat16(), k.bfloat16(), lengths),
        lambda: ga.prompt_attention(q, k, k, lengths, scale=float("inf")),
        lambda: ga.prompt_attention(q.clone().requires_grad_(), k, k, lengths),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"refusal {i} passed")
    with torch.no_grad():
        ga.prompt_attention(q.clone().requires_grad_(), k, k, torch.tensor([0, 3], dtype=i32).cuda())
