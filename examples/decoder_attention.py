#!/usr/bin/env python3
"""Decoder layers with GRINQH linears and the 4-bit key/value cache, end to end.

A Llama-style stack (RMSNorm, qkv_proj, rotary embedding, attention, o_proj,
RMSNorm, gate_up_proj, SiLU * mul, down_proj) with random weights: the linears
are GRINQH's, everything between qkv_proj and o_proj is ``grinqh.attention``:

* ``prompt``: a packed batch of prompts, ``kv4_store`` and ``prompt_attention``;
* ``step``: one token per sequence, ``kv4_store`` and ``kv4_attention``, over all pages or over the ``select`` pages per
  sequence and head that ``kv4_select`` picks by the summaries that ``kv4_summarize`` keeps;
* ``extend``: several more tokens per sequence behind the cached ones, ``kv4_store`` and ``kv4_chunk_attention``.

Room for the tokens is found on the GPU (``kv4_append``): no step waits for the host to know a length.

    python examples/decoder_attention.py          # a small model, a few steps, tokens/s
"""
from __future__ import annotations

import os
import sys
import time

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "vllm-grinqh-plugin_amd"))

import grinqh.kernel  # noqa: E402,F401  (registers torch.ops.grinqh)
from grinqh import attention as ga  # noqa: E402
from grinqh.producer import rmsnorm_sigma, silu_mul_sigma  # noqa: E402
from grinqh.utils import prepare_weight  # noqa: E402

BITS, GROUP = 8, 128


class Linear:
    """A GRINQH linear with random 8-bit weights of a size that keeps activations near one."""

    def __init__(self, k: int, n: int, generator: torch.Generator, thresholds=(0.0, 0.4, 0.9, 1.6)):
        w = torch.randint(-127, 128, (k, n), generator=generator, device="cuda", dtype=torch.int32).to(torch.int8)
        self.planes = prepare_weight(w, BITS)
        self.scale = torch.full((k // GROUP, n), k ** -0.5 / 73.0, dtype=torch.float16, device="cuda")
        self.n, self.thresholds = n, list(thresholds)

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        return torch.ops.grinqh.gemm_or_gemv(x, self.planes, self.scale, None, BITS, GROUP, self.n // 4,
                                             self.thresholds)


class Decoder:
    def __init__(self, layers=2, hidden=512, heads=8, kv_heads=2, head_dim=128, ffn=1024, pages=64, page_size=16,
                 key_group=32, max_pages=16, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.d, self.page, self.max_pages = heads, kv_heads, head_dim, page_size, max_pages
        width = (heads + 2 * kv_heads) * head_dim
        self.layers = [{"qkv": Linear(hidden, width, g), "o": Linear(heads * head_dim, hidden, g),
                        "gate_up": Linear(hidden, 2 * ffn, g), "down": Linear(ffn, hidden, g),
                        "cache": ga.kv4_cache(pages, kv_heads, head_dim, page_size, key_group)} for _ in range(layers)]
        for layer in self.layers:
            layer["summary"] = ga.kv4_summary(layer["cache"])
        self.norm = torch.ones(hidden, dtype=torch.float16, device="cuda")
        self.freq = 10000.0 ** (-torch.arange(0, head_dim, 2, device="cuda").float() / head_dim)
        self.free = torch.arange(pages - 1, -1, -1, dtype=torch.int32, device="cuda")
        self.admit(0)

    def admit(self, sequences: int) -> None:
        """A new batch of empty sequences; all pages are free again."""
        self.table = torch.full((sequences, self.max_pages), -1, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device="cuda")
        self.free_count = torch.full((1,), len(self.free), dtype=torch.int32, device="cuda")

    def _room(self, counts: torch.Tensor, tokens: int) -> ga.Appended:
        """Slots, positions and row offsets of ``counts`` new tokens per sequence; ``before`` is what they had."""
        room = ga.kv4_append(self.table, self.lengths, counts, self.free, self.free_count, self.page, tokens)
        self.before, self.lengths, self.free_count = self.lengths, room.lengths, room.free_count
        return room

    def all_have_room(self) -> bool:
        """Whether every token so far found a page; waits for the GPU.  A server that may run out looks at this before it
        hands out results, and makes the step again from ``before`` and its list of free pages when some have come free."""
        pages = (self.lengths + self.page - 1) // self.page
        place = torch.arange(self.max_pages, device="cuda")
        return bool(((self.table >= 0) | (place >= pages.view(-1, 1))).all()) and int(pages.max()) <= self.max_pages

    def _rotate(self, x: torch.Tensor, position: torch.Tensor) -> torch.Tensor:
        angle = position.float().view(-1, 1, 1) * self.freq
        a, b = x.float().chunk(2, -1)
        return torch.cat((a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()), -1).to(x.dtype)

    def _run(self, h: torch.Tensor, room: ga.Appended, attend) -> torch.Tensor:
        position = room.positions
        for layer in self.layers:
            y, _, _ = rmsnorm_sigma(h, self.norm)
            q, k, v = layer["qkv"](y).split((self.heads * self.d, self.kv_heads * self.d, self.kv_heads * self.d), 1)
            q = self._rotate(q.unflatten(1, (self.heads, self.d)), position)
            k = self._rotate(k.unflatten(1, (self.kv_heads, self.d)), position)
            v = v.unflatten(1, (self.kv_heads, self.d))  # a slice of the projection, as it is
            ga.kv4_store(layer["cache"], k, v, room.slots)
            ga.kv4_summarize(layer["cache"], layer["summary"], self.table, self.before, self.lengths)
            h = h + layer["o"](attend(layer, q, k, v).flatten(1))
            y, _, _ = rmsnorm_sigma(h, self.norm)
            y, _ = silu_mul_sigma(layer["gate_up"](y))
            h = h + layer["down"](y)
        return h

    def prompt(self, h: torch.Tensor, lens) -> torch.Tensor:
        """Hidden states of packed prompts (``lens`` tokens each); fills the cache."""
        room = self._room(torch.tensor(lens, dtype=torch.int32, device="cuda"), len(h))
        return self._run(h, room, lambda layer, q, k, v: ga.prompt_attention(q, k, v, room.ends))

    def step(self, h: torch.Tensor, select: int = 0) -> torch.Tensor:
        """One more token per sequence; with ``select`` it sees that many pages of its sequence per head."""
        room = self._room(torch.ones_like(self.lengths), len(h))

        def attend(layer, q, k, v):
            table, lengths = self.table, self.lengths
            if select:
                table, lengths = ga.kv4_select(q, layer["summary"], table, lengths, self.page, select)
            return ga.kv4_attention(q, layer["cache"], table, lengths)
        return self._run(h, room, attend)

    def extend(self, h: torch.Tensor, lens) -> torch.Tensor:
        """``lens`` more tokens per sequence; their keys and values join the cached ones."""
        room = self._room(torch.tensor(lens, dtype=torch.int32, device="cuda"), len(h))
        return self._run(h, room, lambda layer, q, k, v: ga.kv4_chunk_attention(q, layer["cache"], self.table,
                                                                               self.lengths, room.ends))


def main() -> None:
    model = Decoder(layers=4, hidden=4096, heads=32, kv_heads=8, head_dim=128, ffn=14336, pages=640, max_pages=40)
    batch, length, steps = 16, 512, 64
    model.admit(batch)
    hidden = model.norm.numel()
    h = torch.randn((batch * length, hidden), dtype=torch.float16, device="cuda")
    model.prompt(h, [length] * batch)
    h = torch.randn((batch, hidden), dtype=torch.float16, device="cuda")
    model.step(h)
    norm = lambda h: h / h.float().pow(2).mean(-1, keepdim=True).sqrt().half()  # noqa: E731
    drafted = norm(model.extend(h.repeat_interleave(4, 0), [4] * batch))
    for select in (0, 8):
        h = drafted[3::4]
        torch.cuda.synchronize()
        start = time.perf_counter()
        for _ in range(steps // 2):
            h = norm(model.step(h, select))
        torch.cuda.synchronize()
        t = (time.perf_counter() - start) / (steps // 2)
        what = f"{select} pages per head" if select else "all pages"
        assert model.all_have_room()
        print(f"4 layers, batch {batch}, {length} tokens of context, {what}: {t * 1e3:.2f} ms a step (eager)")


if __name__ == "__main__":
    main()
