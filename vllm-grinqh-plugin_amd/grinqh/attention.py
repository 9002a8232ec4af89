"""Attention between the quantized linears: a key/value cache held in 4 bits
and the attention over whole prompts (libgrinqh_hip.so: grinqh_kv4_*,
grinqh_prompt_attention).

A decoder layer runs ``qkv_proj`` (a GRINQH linear), attention, ``o_proj``.
These functions are the middle part: ``prompt_attention`` for prompts,
``kv4_store`` for the new tokens' keys and values, ``kv4_attention`` for the
single tokens that follow and ``kv4_load`` for a later prompt that shares a
cached prefix.  Queries, keys and values may be slices of the fused projection;
all calls only enqueue work on the current stream and can be captured in a HIP
graph.  There is no backward pass and no forward-mode derivative: inputs that
require a gradient while gradients are recorded, or that carry a tangent, are
refused.  No reference counterpart: the reference leaves
attention to vLLM.
"""
from __future__ import annotations

from functools import lru_cache
from typing import Optional, Tuple

import torch
import torch.autograd.forward_ad as forward_ad

from . import _lib
from .kernel import _Workspaces, _dtype_code

HEAD_DIMS = (64, 128, 256)
GROUPS = (32, 64, 128, 256)

# Counters and partial results of split sequences; the linears' workspaces have
# counters of their own at the same place.
_WORKSPACES = _Workspaces()


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


_stream = torch._C._cuda_getCurrentRawStream  # current_stream() without its wrapper object


def _scale(scale: Optional[float], head_dim: int) -> float:
    return head_dim ** -0.5 if scale is None else float(scale)


@lru_cache(maxsize=1024)
def _workspace_bytes(seqs: int, heads: int, kv_heads: int, head_dim: int, capacity: int) -> int:
    """Workspace of this batch and of every smaller one, so that a program which ran its largest batch can capture the
    others: the library's sizes grow with the batch up to the largest that may share its sequences between blocks, and
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
    tokens of its pages ``page_table[s]`` (int32 ``[seqs, width]``).  ``scale`` defaults to head_dim ** -0.5.  A length
    of 0 gives zeros; a length past the table or a page outside the cache NaN."""
    pages, kv_heads, page, d, group = _cache_layout(cache)
    dev, dtype = cache.device, q.dtype
    dt = _dtype_code(dtype)
    q, q_token, q_head = _rows(q, "q", dev, dtype)
    seqs, heads, dq = q.shape
    if dq != d or heads % kv_heads:
        raise ValueError(f"GRINQH: q {tuple(q.shape)} does not match a cache of {kv_heads} heads of {d} channels")
    if page_table.dim() != 2 or page_table.dtype is not torch.int32 or page_table.device != dev or \
            page_table.shape[0] != seqs:
        raise ValueError(f"GRINQH: page_table must be torch.int32 [{seqs}, width] on {dev}, got {page_table.dtype} "
                         f"{list(page_table.shape)} on {page_table.device}")
    table_stride, one = page_table.stride()
    if one != 1:
        page_table = page_table.contiguous()
        table_stride = page_table.stride(0)
    lengths = _index(lengths, "lengths", torch.int32, seqs, dev)
    width = page_table.shape[1]
    out = torch.empty((seqs, heads, d), dtype=dtype, device=dev)
    with _lib.on_device(dev):
        stream = _stream(dev.index)
        nbytes = _workspace_bytes(seqs, heads, kv_heads, d, width * page)
        ws = _WORKSPACES.get(dev, stream, nbytes) if nbytes else None
        _lib.check(_lib.load_library().grinqh_kv4_attention(
            q.data_ptr(), q_token, q_head, seqs, heads, cache.data_ptr(), pages, kv_heads, page, d, group,
            page_table.data_ptr(), table_stride, width, lengths.data_ptr(), _scale(scale, d), out.data_ptr(), dt,
            ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0, stream),
            "grinqh_kv4_attention")
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
