#!/usr/bin/env python3
"""Decoder layers with GRINQH linears and the 4-bit key/value cache, end to end.

A Llama-style stack (RMSNorm, qkv_proj, rotary embedding, attention, o_proj,
RMSNorm, gate_up_proj, SiLU * mul, down_proj) with random weights: the linears
are GRINQH's, everything between qkv_proj and o_proj is ``grinqh.attention``:

* ``prompt``: a packed batch of prompts, ``kv4_store`` and ``prompt_attention``;
* ``step``: one token per sequence, ``kv4_store`` and ``kv4_attention``;
* ``extend``: more prompt behind a cached prefix, which ``kv4_load`` brings back.

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
        self.norm = torch.ones(hidden, dtype=torch.float16, device="cuda")
        self.freq = 10000.0 ** (-torch.arange(0, head_dim, 2, device="cuda").float() / head_dim)
        self.free = list(range(pages))
        self.table = torch.zeros((0, max_pages), dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(0, dtype=torch.int32, device="cuda")

    def admit(self, sequences: int) -> None:
        """Room for new sequences: max_pages pages each, anywhere in the cache."""
        rows = [[self.free.pop() for _ in range(self.max_pages)] for _ in range(sequences)]
        self.table = torch.tensor(rows, dtype=torch.int32, device="cuda")
        self.lengths = torch.zeros(sequences, dtype=torch.int32, device="cuda")

    def _slots(self, sequence: torch.Tensor, position: torch.Tensor) -> torch.Tensor:
        return self.table[sequence, position // self.page].long() * self.page + position % self.page

    def _rotate(self, x: torch.Tensor, position: torch.Tensor) -> torch.Tensor:
        angle = position.float().view(-1, 1, 1) * self.freq
        a, b = x.float().chunk(2, -1)
        return torch.cat((a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos()), -1).to(x.dtype)

    def _run(self, h: torch.Tensor, position: torch.Tensor, slots: torch.Tensor, attend) -> torch.Tensor:
        for layer in self.layers:
            y, _, _ = rmsnorm_sigma(h, self.norm)
            q, k, v = layer["qkv"](y).split((self.heads * self.d, self.kv_heads * self.d, self.kv_heads * self.d), 1)
            q = self._rotate(q.unflatten(1, (self.heads, self.d)), position)
            k = self._rotate(k.unflatten(1, (self.kv_heads, self.d)), position)
            v = v.unflatten(1, (self.kv_heads, self.d))  # a slice of the projection, as it is
            ga.kv4_store(layer["cache"], k, v, slots)
            h = h + layer["o"](attend(layer["cache"], q, k, v).flatten(1))
            y, _, _ = rmsnorm_sigma(h, self.norm)
            y, _ = silu_mul_sigma(layer["gate_up"](y))
            h = h + layer["down"](y)
        return h

    def prompt(self, h: torch.Tensor, lens) -> torch.Tensor:
        """Hidden states of packed prompts (``lens`` tokens each); fills the cache."""
        sequence = torch.repeat_interleave(torch.arange(len(lens)), torch.tensor(lens)).cuda()
        position = torch.cat([torch.arange(n) for n in lens]).cuda()
        ends = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
        self.lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
        return self._run(h, position, self._slots(sequence, position),
                         lambda cache, q, k, v: ga.prompt_attention(q, k, v, ends))

    def step(self, h: torch.Tensor) -> torch.Tensor:
        """One more token per sequence."""
        position = self.lengths.long()
        self.lengths = self.lengths + 1
        slots = self._slots(torch.arange(len(position), device="cuda"), position)
        return self._run(h, position, slots,
                         lambda cache, q, k, v: ga.kv4_attention(q, cache, self.table, self.lengths))

    def extend(self, h: torch.Tensor, lens) -> torch.Tensor:
        """``lens`` more tokens per sequence; their keys and values join the cached ones."""
        before = self.lengths.tolist()
        after = [a + b for a, b in zip(before, lens)]
        span = lambda first, last: torch.cat([torch.arange(a, b) for a, b in zip(first, last)]).cuda()  # noqa: E731
        owner = lambda n: torch.repeat_interleave(torch.arange(len(n)), torch.tensor(n)).cuda()  # noqa: E731
        ends = torch.tensor([[0] + lens, [0] + after]).cumsum(1).to(torch.int32).cuda()
        position = span(before, after)
        every = self._slots(owner(after), span([0] * len(after), after))
        self.lengths = torch.tensor(after, dtype=torch.int32, device="cuda")
        return self._run(h, position, self._slots(owner(lens), position),
                         lambda cache, q, k, v: ga.prompt_attention(q, *ga.kv4_load(cache, every, q.dtype), ends[0],
                                                                    ends[1]))


def main() -> None:
    model = Decoder(layers=4, hidden=4096, heads=32, kv_heads=8, head_dim=128, ffn=14336, pages=640, max_pages=40)
    batch, length, steps = 16, 512, 64
    model.admit(batch)
    hidden = model.norm.numel()
    h = torch.randn((batch * length, hidden), dtype=torch.float16, device="cuda")
    model.prompt(h, [length] * batch)
    h = torch.randn((batch, hidden), dtype=torch.float16, device="cuda")
    model.step(h)
    torch.cuda.synchronize()
    start = time.perf_counter()
    for _ in range(steps):
        h = model.step(h)
        h = h / h.float().pow(2).mean(-1, keepdim=True).sqrt().half()
    torch.cuda.synchronize()
    t = (time.perf_counter() - start) / steps
    print(f"4 layers, batch {batch}, {length} tokens of context: {t * 1e3:.2f} ms a step (eager)")


if __name__ == "__main__":
    main()
