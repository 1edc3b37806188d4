"""One layer's attention, all of it on the GPU: Q4_K projections, the 8-bit
key/value cache, attention over it, and eviction once a sequence holds more than
its budget.

    python examples/attention_block.py

runs TinyLlama-1.1B's layer shapes (2048 wide, 32 heads of 64 over 4 kv heads)
with synthetic weights: prompts of unequal lengths in pieces, then tokens of all
sequences at once, the decode step as one captured graph. Positions enter as a
distance bias; a model that rotates its queries and keys does so between their
projections and the append, with the rows at positions past[b] + i.
"""
from __future__ import annotations

import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

from rocknpu_amd import hip, kv, synth  # noqa: E402

Q4_K = 4
DECODE_ROWS = 16  # up to here the decode GEMV on the raw rows, above the W8A8 GEMM


class AttentionBlock:
    """`weights` maps q, k, v and o to (Q4_K bytes on the device, rows); `cache`
    is the layer's. Positions enter as a distance bias, `slopes` [heads]."""

    def __init__(self, weights: dict, width: int, heads: int, cache: kv.Cache, slopes: torch.Tensor | None = None):
        self.width, self.heads, self.cache, self.slopes = width, heads, cache, slopes
        self.raw = weights
        inputs = {"q": width, "k": width, "v": width, "o": heads * cache.head_dim}
        self.inputs = inputs
        self.w8 = {name: hip.repack_w8(Q4_K, w, inputs[name], n) for name, (w, n) in weights.items()}
        self.spare = torch.empty_like(cache.dropped)

    def project(self, names, x: torch.Tensor) -> list[torch.Tensor]:
        k = self.inputs[names[0]]
        if x.shape[0] <= DECODE_ROWS:
            return hip.gemv_q_f32(Q4_K, [self.raw[n][0] for n in names], k, [self.raw[n][1] for n in names], x)
        return [hip.matmul_w8a8_f32(x, *self.w8[n], k=k) for n in names]

    def step(self, x: torch.Tensor, past: torch.Tensor, cu: torch.Tensor, max_new: int, max_tokens: int = 0) -> torch.Tensor:
        """x [rows, width] f32: rows cu[b] .. cu[b + 1] - 1 are sequence b's next, behind past[b] tokens."""
        c, rows = self.cache, x.shape[0]
        q, k, v = self.project(("q", "k", "v"), x)
        kv.append(c, k.view(rows, c.kv_heads, c.head_dim), v.view(rows, c.kv_heads, c.head_dim), past, cu, max_new)
        weigh = c.weights is not None and max_new * (self.heads // c.kv_heads) <= kv.MAX_WEIGHT_ROWS
        out = kv.attention(c, q.view(rows, self.heads, c.head_dim), past, cu, max_new, max_tokens=max_tokens,
                           slopes=self.slopes, weights_out=c.weights if weigh else None)
        return self.project(("o",), out.view(rows, -1))[0]

    def trim(self, tokens: torch.Tensor, budget: int, sinks: int = 1, recent: int = 4) -> None:
        """Cuts sequences of tokens [batch] to `budget` blocks; the evicted blocks' pages are their next ones."""
        c = self.cache
        kv.evict(c.table, c.starts, c.weights, tokens, c.dropped, budget, sinks=sinks, recent=recent,
                 out=(c.table, c.starts, c.weights, self.spare))
        c.dropped.copy_(self.spare)


def tinyllama_block(batch: int, max_blocks: int, device="cuda", layer: int = 0) -> AttentionBlock:
    shapes = {name: (i, n) for i, (name, _, n, _) in enumerate(synth.TINYLLAMA_LAYER) if name in "qkvo"}
    weights = {name: (torch.from_numpy(synth.q4_k(n, 2048, layer * len(synth.TINYLLAMA_LAYER) + i)).to(device), n)
               for name, (i, n) in shapes.items()}
    slopes = 2.0 ** -torch.linspace(1, 8, 32, device=device)
    return AttentionBlock(weights, 2048, 32, kv.Cache.empty(batch, 4, 64, max_blocks, device=device), slopes)


def main() -> None:
    dev = torch.device("cuda", 0)
    prompts, piece, tokens, budget, every = [1500, 700, 45, 1], 256, 160, 24, 32
    batch = len(prompts)
    block = tinyllama_block(batch, 64, dev)
    g = torch.Generator(device=dev).manual_seed(1)

    def rows(n):
        return 0.02 * torch.randn((n, block.width), generator=g, device=dev)

    done = [0] * batch
    while done != prompts:
        new = [min(piece, p - d) for p, d in zip(prompts, done)]
        cu = torch.tensor([sum(new[:b]) for b in range(batch + 1)], dtype=torch.int32, device=dev)
        block.step(rows(sum(new)), torch.tensor(done, dtype=torch.int32, device=dev), cu, max(new))
        done = [d + n for d, n in zip(done, new)]

    # a token of every sequence a step: the lengths live on the device, so one graph serves all steps
    past = torch.tensor(done, dtype=torch.int32, device=dev)
    cu = torch.arange(batch + 1, dtype=torch.int32, device=dev)
    x, out = rows(batch), torch.empty((batch, block.width), device=dev)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()

    def decode():
        out.copy_(block.step(x, past, cu, 1))
        past.add_(1)

    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        decode()  # makes the stream's workspaces
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            decode()
        start = time.perf_counter()
        for i in range(1, tokens):
            x.copy_(rows(batch))
            graph.replay()
            if i % every == 0:
                block.trim(past, budget)
        stream.synchronize()
        took = time.perf_counter() - start
    held = [-(-t // kv.BLOCK) - d for t, d in zip(past.tolist(), block.cache.dropped.tolist())]
    print(f"tokens {past.tolist()}, blocks held {held} of a budget of {budget}, outputs finite: "
          f"{bool(torch.isfinite(out).all())}, {took / (tokens - 1) * 1e6:.0f} us a step")


if __name__ == "__main__":
    main()
