"""Attention between the quantized linears: a key/value cache held in 4 bits
and the attention over whole prompts (libgrinqh_hip.so: grinqh_kv4_*,
grinqh_prompt_attention).

A decoder layer runs ``qkv_proj`` (a GRINQH linear), attention, ``o_proj``.
These functions are the middle part: ``prompt_attention`` for prompts,
``kv4_store`` for the new tokens' keys and values, ``kv4_attention`` for the
single tokens that follow, ``kv4_chunk_attention`` for several new tokens per
sequence behind cached ones, and ``kv4_load`` for reading back.  Once per step,
``kv4_append`` finds room for the new tokens.  For long contexts
``kv4_summarize`` keeps the mean key of every page and ``kv4_select`` picks the
pages that ``kv4_attention`` then reads.  Queries, keys and values may be slices of the fused projection;
all calls only enqueue work on the current stream and can be captured in a HIP
graph.  There is no backward pass and no forward-mode derivative: inputs that
require a gradient while gradients are recorded, or that carry a tangent, are
refused.  No reference counterpart: the reference leaves
attention to vLLM.
"""
from __future__ import annotations

import threading
from functools import lru_cache
from typing import NamedTuple, Optional, Tuple

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib
from .kernel import _Workspaces, _dtype_code

HEAD_DIMS = (64, 128, 256)
GROUPS = (32, 64, 128, 256)

# Counters and partial results of split sequences; the linears' workspaces have
# counters of their own at the same place.
_WORKSPACES = _Workspaces()


class _GraphWorkspaces:
    """Workspaces of captured calls, in the graph's own memory, so that graphs which were captured on one stream may be
    replayed at the same time on several: one for all calls of a capture on a stream, which follow each other.  The
    counters are cleared once in every replay, in front of the first call; every call leaves them zero.  Kept here until
    the stream's next capture, as the memory must not be given to anything between two calls of a graph."""

    def __init__(self):
        self._bufs = {}  # (device, stream) -> (capture, buffer)
        self._lock = threading.Lock()

    def get(self, device: torch.device, stream: int, nbytes: int) -> torch.Tensor:
        key, capture = (device.index, stream), _lib.load_library().grinqh_capture_id(stream)
        with self._lock:
            before, ws = self._bufs.get(key, (0, None))
            if before != capture or capture == 0 or ws.numel() < nbytes:
                ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
                ws[:_lib.KV4_COUNTER_BYTES].zero_()
                self._bufs[key] = capture, ws
            return ws


_GRAPH_WORKSPACES = _GraphWorkspaces()


def _workspace(device: torch.device, stream: int, nbytes: int) -> Optional[torch.Tensor]:
    """The stream's workspace, or the graph's that is being captured; for the current device"""
    if nbytes == 0:
        return None
    return (_GRAPH_WORKSPACES if torch.cuda.is_current_stream_capturing() else _WORKSPACES).get(device, stream, nbytes)


def kv4_record_bytes(head_dim: int, group: Optional[int] = None) -> int:
    """Bytes of 16 tokens of one head, keys and values (include/grinqh.h describes the layout)."""
    group = head_dim if group is None else group
    if head_dim not in HEAD_DIMS or group not in GROUPS or group > head_dim:
        raise ValueError(f"GRINQH: head_dim must be one of {HEAD_DIMS} and group one of {GROUPS}, at most head_dim; "
                         f"got {head_dim}, {group}")
    return 16 * head_dim + 64 * (head_dim // group + 1)


def kv4_cache(pages: int, kv_heads: int, head_dim: int, page_size: int = 16, group: Optional[int] = None,
              device="cuda") -> torch.Tensor:
    """An empty cache: uint8 ``[pages, kv_heads, page_size / 16, record]``.
    ``group`` channels share a key's scale (default: the whole head); outlier
    channels of the keys then cost only their own group's accuracy."""
    if page_size < 16 or page_size & (page_size - 1):
        raise ValueError(f"GRINQH: page_size must be a power of two of at least 16, got {page_size}")
    if pages < 0 or kv_heads <= 0:
        raise ValueError(f"GRINQH: a cache has pages >= 0 and kv_heads > 0, got {pages}, {kv_heads}")
    return torch.zeros((pages, kv_heads, page_size // 16, kv4_record_bytes(head_dim, group)), dtype=torch.uint8,
                       device=device)


# The largest batch whose sequences may be shared by several blocks, in sequences
# and in pairs of a sequence and up to 16 query heads of one key/value head.
_SHARED_SEQS = 1024
_SHARED_UNITS = 1 << 15

_LAYOUTS = {kv4_record_bytes(d, g): (d, g) for d in HEAD_DIMS for g in GROUPS if g <= d}


def _cache_layout(cache: torch.Tensor) -> Tuple[int, int, int, int, int]:
    """(pages, kv_heads, page_size, head_dim, group) of a cache tensor"""
    if not cache.is_cuda:
        raise ValueError("GRINQH: the cache must be on a HIP device; there is no CPU path")
    shape = cache.shape
    layout = _LAYOUTS.get(shape[3]) if len(shape) == 4 else None
    if layout is None or shape[1] == 0 or cache.dtype is not torch.uint8 or not cache.is_contiguous():
        raise ValueError("GRINQH: a cache is a contiguous uint8 tensor [pages, kv_heads > 0, page_size / 16, record] "
                         f"(kv4_cache), got {cache.dtype} {tuple(shape)}")
    return shape[0], shape[1], 16 * shape[2], layout[0], layout[1]


def _rows(x: torch.Tensor, name: str, device: torch.device, dtype: torch.dtype,
          least: int = 0) -> Tuple[torch.Tensor, int, int]:
    """x [tokens, heads, head_dim] as the kernels read it (16-byte aligned rows, distances multiples of 8, tokens at
    least ``least`` apart; copied where it is not), and its token and head distances"""
    if x.device != device or x.dtype is not dtype:
        raise ValueError(f"GRINQH: {name} must be {dtype} on {device}, got {x.dtype} on {x.device}")
    if x.requires_grad and torch.is_grad_enabled():
        raise ValueError(f"GRINQH: {name} requires a gradient; the attention operators have no backward pass")
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(x).tangent is not None:
        raise ValueError(f"GRINQH: {name} has a tangent; the attention operators have no forward-mode derivative")
    stride = x.stride()
    if len(stride) != 3:
        raise ValueError(f"GRINQH: {name} must be [tokens, heads, head_dim], got {tuple(x.shape)}")
    t, h, c = stride
    if c != 1 or t % 8 or h % 8 or t < least or t > 1 << 23 or h > 1 << 23 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)  # contiguous() keeps what only lies askew
        t, h, c = x.stride()
    return x, t, h


def _index(x: torch.Tensor, name: str, dtype: torch.dtype, n: int, device: torch.device) -> torch.Tensor:
    if x.device != device or x.dtype is not dtype or x.dim() != 1 or x.shape[0] != n:
        raise ValueError(f"GRINQH: {name} must be {dtype} [{n}] on {device}, got {x.dtype} {list(x.shape)} on "
                         f"{x.device}")
    return x if x.is_contiguous() else x.contiguous()


def _table(x: torch.Tensor, seqs: int, device: torch.device) -> Tuple[torch.Tensor, int]:
    """A page table [seqs, width] and the distance of its rows"""
    if x.dim() != 2 or x.dtype is not torch.int32 or x.device != device or x.shape[0] != seqs:
        raise ValueError(f"GRINQH: page_table must be torch.int32 [{seqs}, width] on {device}, got {x.dtype} "
                         f"{list(x.shape)} on {x.device}")
    stride, one = x.stride()
    if one != 1:
        x = x.contiguous()
        stride = x.stride(0)
    return x, stride


def _head_table(x: torch.Tensor, seqs: int, kv_heads: int, device: torch.device) -> Tuple[torch.Tensor, int, int]:
    """A page table [seqs, kv_heads, width] and the distances of its sequences and heads"""
    if x.dtype is not torch.int32 or x.device != device or x.shape[:2] != (seqs, kv_heads):
        raise ValueError(f"GRINQH: page_table must be torch.int32 [{seqs}, {kv_heads}, width] on {device}, got {x.dtype} "
                         f"{list(x.shape)} on {x.device}")
    if x.stride(2) != 1:
        x = x.contiguous()
    return x, x.stride(0), x.stride(1)


_stream = torch._C._cuda_getCurrentRawStream  # current_stream() without its wrapper object


def _scale(scale: Optional[float], head_dim: int) -> float:
    return head_dim ** -0.5 if scale is None else float(scale)


@lru_cache(maxsize=1024)
def _workspace_bytes(seqs: int, heads: int, kv_heads: int, head_dim: int, capacity: int) -> int:
    """Workspace of this batch and of every smaller one, so that batches of changing size need no larger one: the
    library's sizes grow with the batch up to the largest that may share its sequences between blocks, and
    are 0 beyond."""
    tiles = kv_heads * -(-(heads // kv_heads) // 16)
    seqs = min(seqs, _SHARED_SEQS, _SHARED_UNITS // tiles) if heads >= kv_heads else seqs
    return _lib.load_library().grinqh_kv4_attention_workspace_bytes(seqs, heads, kv_heads, head_dim, capacity)


def kv4_store(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
    """Write keys and values ``[tokens, kv_heads, head_dim]`` at ``slots`` (int64 ``[tokens]``: page * page_size +
    place).  Slots outside the cache (-1: padding) are skipped; no two tokens may have the same slot."""
    pages, heads, page, d, group = _cache_layout(cache)
    dev, dtype = cache.device, k.dtype
    dt = _dtype_code(dtype)
    k, k_token, k_head = _rows(k, "k", dev, dtype)
    v, v_token, v_head = _rows(v, "v", dev, dtype)
    n = k.shape[0]
    if k.shape != (n, heads, d) or v.shape != k.shape:
        raise ValueError(f"GRINQH: k and v must be [tokens, {heads}, {d}] for this cache, got {tuple(k.shape)} and "
                         f"{tuple(v.shape)}")
    slots = _index(slots, "slots", torch.int64, n, dev)
    with _lib.on_device(dev):
        _lib.check(_lib.load_library().grinqh_kv4_store(
            k.data_ptr(), k_token, k_head, v.data_ptr(), v_token, v_head, slots.data_ptr(), n, cache.data_ptr(), pages,
            heads, page, d, group, dt, _stream(dev.index)), "grinqh_kv4_store")


def kv4_load(cache: torch.Tensor, slots: torch.Tensor, dtype: torch.dtype = torch.float16,
             ) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values ``[tokens, kv_heads, head_dim]`` of ``slots``; slots outside the cache give zeros."""
    pages, heads, page, d, group = _cache_layout(cache)
    dev = cache.device
    dt = _dtype_code(dtype)
    n = slots.numel()
    slots = _index(slots, "slots", torch.int64, n, dev)
    k = torch.empty((n, heads, d), dtype=dtype, device=dev)
    v = torch.empty_like(k)
    with _lib.on_device(dev):
        _lib.check(_lib.load_library().grinqh_kv4_load(
            cache.data_ptr(), pages, heads, page, d, group, slots.data_ptr(), n, k.data_ptr(), v.data_ptr(), dt,
            _stream(dev.index)), "grinqh_kv4_load")
    return k, v


def kv4_attention(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                  scale: Optional[float] = None) -> torch.Tensor:
    """Attention of one query token per sequence, ``q [seqs, heads, head_dim]``, over the first ``lengths[s]`` (int32)
    tokens of its pages ``page_table[s]`` (int32 ``[seqs, width]``, or ``[seqs, kv_heads, width]``: a choice of pages
    per key/value head, as ``kv4_select`` makes it).  ``scale`` defaults to head_dim ** -0.5.  A length of 0 gives
    zeros; a length past the table or a page outside the cache NaN."""
    pages, kv_heads, page, d, group = _cache_layout(cache)
    dev, dtype = cache.device, q.dtype
    dt = _dtype_code(dtype)
    q, q_token, q_head = _rows(q, "q", dev, dtype)
    seqs, heads, dq = q.shape
    if dq != d or heads % kv_heads:
        raise ValueError(f"GRINQH: q {tuple(q.shape)} does not match a cache of {kv_heads} heads of {d} channels")
    if page_table.dim() == 3:
        page_table, table_stride, table_head = _head_table(page_table, seqs, kv_heads, dev)
    else:
        page_table, table_stride = _table(page_table, seqs, dev)
        table_head = None
    lengths = _index(lengths, "lengths", torch.int32, seqs, dev)
    width = page_table.shape[-1]
    out = torch.empty((seqs, heads, d), dtype=dtype, device=dev)
    with _lib.on_device(dev):
        stream = _stream(dev.index)
        nbytes = _workspace_bytes(seqs, heads, kv_heads, d, width * page)
        ws = _workspace(dev, stream, nbytes)
        at, room = (ws.data_ptr(), ws.numel()) if ws is not None else (None, 0)
        if table_head is None:
            _lib.check(_lib.load_library().grinqh_kv4_attention(
                q.data_ptr(), q_token, q_head, seqs, heads, cache.data_ptr(), pages, kv_heads, page, d, group,
                page_table.data_ptr(), table_stride, width, lengths.data_ptr(), _scale(scale, d), out.data_ptr(), dt,
                at, room, stream), "grinqh_kv4_attention")
        else:
            _lib.check(_lib.load_library().grinqh_kv4_attention_selected(
                q.data_ptr(), q_token, q_head, seqs, heads, cache.data_ptr(), pages, kv_heads, page, d, group,
                page_table.data_ptr(), table_stride, table_head, width, lengths.data_ptr(), _scale(scale, d),
                out.data_ptr(), dt, at, room, stream), "grinqh_kv4_attention_selected")
    return out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, ends: torch.Tensor,
                     key_ends: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention over packed sequences: ``q [tokens, heads, head_dim]``, ``k`` and ``v [keys, kv_heads,
    head_dim]``.  Sequence s has rows ``ends[s] .. ends[s + 1] - 1`` (int32 ``[seqs + 1]``, ascending) and keys
    ``key_ends[s] .. key_ends[s + 1] - 1`` (default: as its rows); its last row sees all its keys, the row before one
    fewer, and so on.  Rows that see no key, or lie in front of the first sequence or behind the last, give zeros.
    ``scale`` defaults to head_dim ** -0.5."""
    dev, dtype = q.device, q.dtype
    if not q.is_cuda:
        raise ValueError(f"GRINQH: q must be on a HIP device (got {dev}); there is no CPU path")
    dt = _dtype_code(dtype)
    q, q_token, q_head = _rows(q, "q", dev, dtype)
    tokens, heads, d = q.shape
    k, k_token, k_head = _rows(k, "k", dev, dtype, d)  # not broadcast, not overlapping
    v, v_token, v_head = _rows(v, "v", dev, dtype, d)
    keys, kv_heads, dk = k.shape
    if d not in HEAD_DIMS or dk != d or v.shape != k.shape or kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError(f"GRINQH: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not fit: head_dim "
                         f"must be one of {HEAD_DIMS}, the heads a multiple of the key/value heads")
    seqs = ends.numel() - 1
    if seqs < 0:
        raise ValueError(f"GRINQH: ends must be int32 [seqs + 1], got {list(ends.shape)}")
    ends = _index(ends, "ends", torch.int32, seqs + 1, dev)
    if key_ends is None:
        if keys != tokens:
            raise ValueError(f"GRINQH: {keys} keys for {tokens} rows need key_ends")
        key_ends = ends
    else:
        key_ends = _index(key_ends, "key_ends", torch.int32, seqs + 1, dev)
    out = torch.empty((tokens, heads, d), dtype=dtype, device=dev)
    with _lib.on_device(dev):
        _lib.check(_lib.load_library().grinqh_prompt_attention(
            q.data_ptr(), q_token, q_head, k.data_ptr(), k_token, k_head, v.data_ptr(), v_token, v_head,
            ends.data_ptr(), key_ends.data_ptr(), seqs, tokens, keys, heads, kv_heads, d, _scale(scale, d),
            out.data_ptr(), dt, _stream(dev.index)), "grinqh_prompt_attention")
    return out


class Appended(NamedTuple):
    """What ``kv4_append`` found: for the rows of the batch, for its sequences and for the list of free pages."""
    slots: torch.Tensor       # int64 [tokens], for kv4_store; -1: none
    positions: torch.Tensor   # int32 [tokens]: place in the sequence; 0 behind the last one
    ends: torch.Tensor        # int32 [seqs + 1]: sequence s has rows ends[s] .. ends[s + 1] - 1
    lengths: torch.Tensor     # int32 [seqs], the new tokens counted
    free_count: torch.Tensor  # int32 [1]


def kv4_append(page_table: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor, free: torch.Tensor,
               free_count: torch.Tensor, page_size: int, tokens: int) -> Appended:
    """Room for ``counts[s]`` (int32 ``[seqs]``) new tokens of sequences that hold ``lengths[s]``, without the host
    knowing either.  The pages they need beyond those they have come from the end of ``free[:free_count]`` (int32;
    ``free_count [1]``), in the order of the sequences, and are written into ``page_table`` (int32 ``[seqs, width]``) in
    place; nothing else that is given changes.  ``tokens`` is the number of rows of the batch's buffers, the new tokens
    packed in front: rows behind the last sequence have slot -1, tokens that do not fit are not counted.  Where pages
    run out the table gets -1, and where it ends nothing: such tokens have slot -1 (``kv4_store`` skips them) and the
    attention of their sequences is NaN.  They are counted in the lengths, and later calls do not look for their pages
    again: a slot of -1 in front of row ``ends[-1]`` says so.  The call is then made again from the lengths and the list
    that it was given, which it has not changed, with fewer tokens or when pages have been put behind that list; it writes
    the same entries of the table anew."""
    dev = page_table.device
    if not page_table.is_cuda:
        raise ValueError(f"GRINQH: page_table must be on a HIP device (got {dev}); there is no CPU path")
    seqs = lengths.shape[0] if lengths.dim() == 1 else -1
    lengths = _index(lengths, "lengths", torch.int32, seqs, dev)
    table, table_stride = _table(page_table, seqs, dev)
    width = table.shape[1]
    if table is not page_table or seqs > 1 and table_stride < width:
        raise ValueError("GRINQH: page_table is written in place: its rows must be contiguous and must not overlap, got "
                         f"strides {page_table.stride()}")
    table_stride = max(table_stride, width)
    counts = _index(counts, "counts", torch.int32, seqs, dev)
    free = _index(free, "free", torch.int32, free.numel(), dev)
    free_count = _index(free_count, "free_count", torch.int32, 1, dev)
    if page_size < 16 or page_size & (page_size - 1) or not 0 <= tokens < 1 << 23:
        raise ValueError(f"GRINQH: page_size must be a power of two of at least 16, tokens from 0 to 2^23 - 1; got "
                         f"{page_size}, {tokens}")
    slots = torch.empty(tokens, dtype=torch.int64, device=dev)
    positions, ends, after, count = torch.empty(
        tokens + 2 * seqs + 2, dtype=torch.int32, device=dev).split((tokens, seqs + 1, seqs, 1))
    with _lib.on_device(dev):
        _lib.check(_lib.load_library().grinqh_kv4_append(
            table.data_ptr(), table_stride, width, page_size, lengths.data_ptr(), counts.data_ptr(), seqs,
            free.data_ptr(), free.shape[0], free_count.data_ptr(), tokens, slots.data_ptr(), positions.data_ptr(),
            ends.data_ptr(), after.data_ptr(), count.data_ptr(), _stream(dev.index)), "grinqh_kv4_append")
    return Appended(slots, positions, ends, after, count)


def kv4_chunk_attention(q: torch.Tensor, cache: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                        ends: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention of several new tokens per sequence, which the cache holds already: ``q [tokens, heads,
    head_dim]``, sequence s has rows ``ends[s] .. ends[s + 1] - 1`` (int32 ``[seqs + 1]``, ascending) and the first
    ``lengths[s]`` (int32) tokens of its pages ``page_table[s]`` (int32 ``[seqs, width]``).  Its last row sees all of
    them, the row before one fewer, and so on.  Rows that see none, in front of the first sequence or behind the last
    give zeros; a length past the table makes the sequence's rows NaN, a page outside the cache those that see it (and
    perhaps others of the sequence).  ``scale`` defaults to head_dim ** -0.5.  What is beside a sequence in the batch
    may change its results by their roundings; the same call gives the same bits."""
    pages, kv_heads, page, d, group = _cache_layout(cache)
    dev, dtype = cache.device, q.dtype
    dt = _dtype_code(dtype)
    q, q_token, q_head = _rows(q, "q", dev, dtype)
    tokens, heads, dq = q.shape
    if dq != d or heads == 0 or heads % kv_heads:
        raise ValueError(f"GRINQH: q {tuple(q.shape)} does not match a cache of {kv_heads} heads of {d} channels")
    seqs = ends.numel() - 1
    if seqs < 0:
        raise ValueError(f"GRINQH: ends must be int32 [seqs + 1], got {list(ends.shape)}")
    ends = _index(ends, "ends", torch.int32, seqs + 1, dev)
    page_table, table_stride = _table(page_table, seqs, dev)
    lengths = _index(lengths, "lengths", torch.int32, seqs, dev)
    width = page_table.shape[1]
    out = torch.empty((tokens, heads, d), dtype=dtype, device=dev)
    nbytes = _chunk_workspace_bytes(tokens, seqs, heads, kv_heads, d, width * page)
    with _lib.on_device(dev):
        stream = _stream(dev.index)
        ws = _workspace(dev, stream, nbytes)
        _lib.check(_lib.load_library().grinqh_kv4_chunk_attention(
            q.data_ptr(), q_token, q_head, tokens, heads, cache.data_ptr(), pages, kv_heads, page, d, group,
            page_table.data_ptr(), table_stride, width, lengths.data_ptr(), ends.data_ptr(), seqs, _scale(scale, d),
            out.data_ptr(), dt, ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0, stream),
            "grinqh_kv4_chunk_attention")
    return out


@lru_cache(maxsize=1024)
def _chunk_workspace_bytes(tokens: int, seqs: int, heads: int, kv_heads: int, head_dim: int, capacity: int) -> int:
    return _lib.load_library().grinqh_kv4_chunk_attention_workspace_bytes(tokens, seqs, heads, kv_heads, head_dim,
                                                                          capacity)


def kv4_summary(cache: torch.Tensor) -> torch.Tensor:
    """An empty summary of a cache's pages: int8 ``[pages, kv_heads, head_dim + 16]``, of every page and head the mean
    key's codes, their step (float32 in 4 bytes) and 12 unused bytes."""
    pages, kv_heads, _, d, _ = _cache_layout(cache)
    return torch.zeros((pages, kv_heads, d + 16), dtype=torch.int8, device=cache.device)


def _summary_layout(summary: torch.Tensor) -> Tuple[int, int, int]:
    """(pages, kv_heads, head_dim) of a summary"""
    shape = summary.shape
    if not summary.is_cuda:
        raise ValueError("GRINQH: the summary must be on a HIP device; there is no CPU path")
    if len(shape) != 3 or shape[2] - 16 not in HEAD_DIMS or shape[1] == 0 or summary.dtype is not torch.int8 or \
            not summary.is_contiguous():
        raise ValueError("GRINQH: a summary is a contiguous int8 tensor [pages, kv_heads > 0, head_dim + 16] "
                         f"(kv4_summary), got {summary.dtype} {tuple(shape)}")
    return shape[0], shape[1], shape[2] - 16


def kv4_summarize(cache: torch.Tensor, summary: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor,
                  lengths: torch.Tensor) -> None:
    """Bring ``summary`` up to date for every page that tokens ``starts[s] .. lengths[s] - 1`` of a sequence lie in
    (int32 ``[seqs]`` both: the lengths before and after ``kv4_append``; 0 and the lengths for all of their pages).
    Called after ``kv4_store``.  Sequences that share a page must agree on how many of its tokens count.  Sums are exact
    for pages of up to 4096 tokens."""
    pages, kv_heads, page, d, group = _cache_layout(cache)
    dev = cache.device
    if _summary_layout(summary) != (pages, kv_heads, d) or summary.device != dev:
        raise ValueError(f"GRINQH: summary {tuple(summary.shape)} on {summary.device} does not match a cache of {pages} "
                         f"pages, {kv_heads} heads of {d} channels on {dev}")
    seqs = lengths.shape[0] if lengths.dim() == 1 else -1
    lengths = _index(lengths, "lengths", torch.int32, seqs, dev)
    starts = _index(starts, "starts", torch.int32, seqs, dev)
    page_table, table_stride = _table(page_table, seqs, dev)
    with _lib.on_device(dev):
        _lib.check(_lib.load_library().grinqh_kv4_summarize(
            cache.data_ptr(), pages, kv_heads, page, d, group, summary.data_ptr(), page_table.data_ptr(), table_stride,
            page_table.shape[1], starts.data_ptr(), lengths.data_ptr(), seqs, _stream(dev.index)),
            "grinqh_kv4_summarize")


def kv4_select(q: torch.Tensor, summary: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, page_size: int,
               count: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """For one query token per sequence, ``q [seqs, heads, head_dim]``, the ``count`` (at least 2) pages of each
    sequence and key/value head whose mean keys promise the largest logits; the first page and the last are always
    among them.  Returns a page table per head, int32 ``[seqs, kv_heads, count]`` in the order of the sequence (-1 behind
    the last page), and how many tokens the selected pages hold, int32 ``[seqs]``: both as ``kv4_attention`` takes them.
    Scores are exact sums of what the summaries hold, equal ones go to the page that comes first."""
    pages, kv_heads, d = _summary_layout(summary)
    dev, dtype = summary.device, q.dtype
    dt = _dtype_code(dtype)
    q, q_token, q_head = _rows(q, "q", dev, dtype)
    seqs, heads, dq = q.shape
    if dq != d or heads == 0 or heads % kv_heads:
        raise ValueError(f"GRINQH: q {tuple(q.shape)} does not match a summary of {kv_heads} heads of {d} channels")
    if page_size < 16 or page_size & (page_size - 1) or count < 2:
        raise ValueError(f"GRINQH: page_size must be a power of two of at least 16, count at least 2; got {page_size}, "
                         f"{count}")
    page_table, table_stride = _table(page_table, seqs, dev)
    lengths = _index(lengths, "lengths", torch.int32, seqs, dev)
    width = page_table.shape[1]
    selected = torch.empty((seqs, kv_heads, count), dtype=torch.int32, device=dev)
    after = torch.empty(seqs, dtype=torch.int32, device=dev)
    lib = _lib.load_library()
    nbytes = lib.grinqh_kv4_select_workspace_bytes(seqs, kv_heads, width, count)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    with _lib.on_device(dev):
        _lib.check(lib.grinqh_kv4_select(
            q.data_ptr(), q_token, q_head, seqs, heads, summary.data_ptr(), pages, kv_heads, page_size, d,
            page_table.data_ptr(), table_stride, width, lengths.data_ptr(), count, selected.data_ptr(),
            after.data_ptr(), dt, ws.data_ptr() if ws is not None else None, nbytes, _stream(dev.index)),
            "grinqh_kv4_select")
    return selected, after
