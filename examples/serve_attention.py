"""Serving a stack of attention layers with the operators between the matmuls.

Prompts of several lengths are answered together: their tokens go through every
layer at once, then one token a sequence a step, from a CUDA graph.  A layer is

    h, n = rms_norm(y + h)          the residual's addition and the norm
    q, k, v = n W_qkv               an xt matmul program
    cache_append(rope(k), v)        into the paged int8 cache
    y = attention(rope(q)) W_out    an xt matmul program

Run it with ``python examples/serve_attention.py [--layers 2] [--steps 32]``.
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch

import xtile as xt


@xt.kernel
def matmul(lhs, rhs, out, tm, tn, tk, ksteps):
    i, j = xt.bid(0), xt.bid(1)
    acc = None
    for k in range(ksteps):
        p = xt.matmul(xt.load(lhs, index=(i, k), shape=(tm, tk)), xt.load(rhs, index=(k, j), shape=(tk, tn)))
        acc = p if acc is None else acc + p
    xt.store(out, index=(i, j), tile=acc)


ROWS = 128  # the matmul program's tile: arrays of rows are padded to whole ones


class Product:
    """x [rows, n] bf16 times w [n, m] bf16 to f32, one traced program for each number of rows."""

    def __init__(self, w) -> None:
        self.w, self.programs = w, {}

    def __call__(self, x, out):
        rows, (n, m) = x.shape[0], self.w.shape
        if rows not in self.programs:
            a = xt.Array
            self.programs[rows] = xt.convert(
                matmul, args=(a((rows, n), xt.bfloat16), a((n, m), xt.bfloat16), a((rows, m), xt.float32), ROWS, 128, 64, n // 64),
                grid=(rows // ROWS, m // 128, 1))
        xt.launch(self.programs[rows], x, self.w, out)
        return out


class Layer:
    def __init__(self, gen, width, q_heads, kv_heads, dim, pages, device) -> None:
        def weights(n, m):
            return (torch.randn(n, m, generator=gen) / n ** 0.5).to(device, torch.bfloat16)

        self.q_heads, self.kv_heads, self.dim = q_heads, kv_heads, dim
        self.norm = (1 + 0.1 * torch.randn(width, generator=gen)).to(device)
        self.qkv = Product(weights(width, (q_heads + 2 * kv_heads) * dim))
        self.out = Product(weights(q_heads * dim, width))
        self.cache = xt.KVCache.empty(pages, kv_heads, dim, device=device)


class Batch:
    """The new tokens of a step: where they stand, and the buffers they pass through."""

    def __init__(self, layer, starts, lengths, pages, tokens, most, device) -> None:
        self.starts, self.lengths, self.pages, self.tokens, self.most = starts, lengths, pages, tokens, most
        rows = -(-tokens // ROWS) * ROWS
        width, heads, dim = layer.norm.shape[0], layer.q_heads, layer.dim
        self.positions = torch.empty(tokens, dtype=torch.int32, device=device)
        self.h = torch.zeros(rows, width, device=device)
        self.y = torch.zeros(rows, width, device=device)
        self.n = torch.zeros(rows, width, dtype=torch.bfloat16, device=device)
        self.qkv = torch.zeros(rows, heads + 2 * layer.kv_heads, dim, device=device)
        self.q = torch.empty(tokens, heads, dim, dtype=torch.bfloat16, device=device)
        self.seen = torch.zeros(rows, heads, dim, dtype=torch.bfloat16, device=device)


def step(layers, table, batch, x):
    """The batch's tokens x [tokens, width] through every layer: what the last one adds to them, and the sum."""
    t = batch.tokens
    batch.h.zero_()
    batch.y[:t] = x
    for layer in layers:
        xt.rms_norm(batch.y, layer.norm, batch.n, residual=batch.h, residual_out=batch.h)
        layer.qkv(batch.n, batch.qkv.view(batch.qkv.shape[0], -1))
        q, k, v = batch.qkv[:t].split([layer.q_heads, layer.kv_heads, layer.kv_heads], dim=1)
        xt.rope(q, batch.positions, table, batch.q)
        xt.cache_append(layer.cache, k, v, batch.starts, batch.lengths, batch.pages, rope=table)
        xt.cache_attention(layer.cache, batch.q, batch.starts, batch.lengths, batch.pages, batch.seen[:t], max_new=batch.most)
        layer.out(batch.seen.view(batch.seen.shape[0], -1), batch.y)
    return batch.h[:t] + batch.y[:t]


class Server:
    def __init__(self, prompts, steps, *, layers=2, width=1024, q_heads=8, kv_heads=2, dim=128, seed=0, device="cuda") -> None:
        gen = torch.Generator().manual_seed(seed)
        self.prompts, self.steps, self.device = prompts, steps, device
        page, seqs = 64, len(prompts)
        need = [-(-(n + steps) // page) for n in prompts]
        order = torch.randperm(sum(need), generator=gen).to(torch.int32)
        pages = torch.zeros(seqs, max(need), dtype=torch.int32)
        for b, part in enumerate(order.split(need)):
            pages[b, :need[b]] = part
        self.pages = pages.to(device)
        self.layers = [Layer(gen, width, q_heads, kv_heads, dim, sum(need), device) for _ in range(layers)]
        self.table = xt.RopeTable.build(max(prompts) + steps, dim, device=device)
        self.lengths = torch.tensor(prompts, dtype=torch.int32, device=device)
        starts = torch.tensor([0] + prompts, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(device)
        self.prompt = Batch(self.layers[0], starts, self.lengths, self.pages, sum(prompts), max(prompts), device)
        self.prompt.positions.copy_(torch.cat([torch.arange(n, dtype=torch.int32) for n in prompts]))
        ones = torch.arange(seqs + 1, dtype=torch.int32, device=device)
        self.single = Batch(self.layers[0], ones, self.lengths, self.pages, seqs, 1, device)
        self.x = torch.empty(seqs, width, device=device)
        self.result = torch.empty(seqs, width, device=device)
        self.graph = None

    def prefill(self, x):
        return step(self.layers, self.table, self.prompt, x)

    def _decode(self):
        self.single.positions.copy_(self.lengths)  # the new token's position
        self.lengths += 1
        self.result.copy_(step(self.layers, self.table, self.single, self.x))

    def decode(self, x):
        """One more token of every sequence; x is valid until the next call."""
        self.x.copy_(x)
        if self.graph is None:
            # run once for real, and once more to record it, which computes nothing
            self._decode()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self._decode()
        else:
            self.graph.replay()
        return self.result

    def cached(self, layer, sequence, length):
        """The keys and values that a sequence holds in a layer, as numbers: [length, kv_heads, dim] each."""
        cache, pages = self.layers[layer].cache, self.pages[sequence].long()
        keys = xt.dequantize(cache.k[pages], cache.k_scale[pages], dtype=torch.float32)
        values = xt.dequantize(cache.v[pages], cache.v_scale[pages], dtype=torch.float32)
        return [t.transpose(1, 2).reshape(-1, cache.heads, cache.dim)[:length] for t in (keys, values)]


def raise_for_device_error() -> None:
    code = xt.device_error()  # which clears it
    if code:
        raise RuntimeError(f"a kernel reported {code:#x}")


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--prompts", type=int, nargs="+", default=[700, 33, 1500, 256])
    a = ap.parse_args()
    server = Server(a.prompts, a.steps, layers=a.layers)
    width = server.x.shape[1]
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(sum(a.prompts), width, generator=gen, device="cuda")
    events = [torch.cuda.Event(enable_timing=True) for _ in range(4)]
    server.prefill(x)  # traces the programs; the lengths stay, so the next call stores the same tokens again
    events[0].record()
    y = server.prefill(x)
    events[1].record()
    last = y[torch.tensor(a.prompts).cumsum(0).cuda() - 1]
    last = server.decode(last).clone()
    events[2].record()
    for _ in range(a.steps - 1):
        last = server.decode(last)
    events[3].record()
    torch.cuda.synchronize()
    raise_for_device_error()
    print(f"{sum(a.prompts)} prompt tokens: {events[0].elapsed_time(events[1]):.3f} ms")
    if a.steps > 1:
        print(f"{len(a.prompts)} tokens a step: {events[2].elapsed_time(events[3]) / (a.steps - 1) * 1e3:.1f} us")


if __name__ == "__main__":
    main()
