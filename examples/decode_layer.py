"""One decoder layer that decodes with 8-bit activations, 4-bit weights and a
4-bit paged key/value cache, made of the package's own ops:

    add + RMS norm -> int8          add_rmsnorm_quant
    q, k, v projection              w4_matmul (int8 rows, 4-bit weights)
    rotary embedding                rope
    cache                           kv_cache_write, cache_attention
    output projection               w4_matmul
    add + RMS norm -> int8          add_rmsnorm_quant
    gate and up projection          w4_matmul
    SwiGLU                          swiglu
    down projection                 w4_matmul

    python examples/decode_layer.py                # 4096 wide, FFN 11008, on one B200
    python examples/decode_layer.py --batch 64 --context 4096 --steps 32

It fills the cache with a prompt of random keys and values, decodes `steps`
tokens per sequence with the step captured in a CUDA graph, compares the last
one with the same layer in float32 and prints the time per step.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "ouroboros-kernelsmith_b200"))

import b200k  # noqa: E402


class DecoderLayer:
    """Random weights of a layer, its cache and the pages of `batch` sequences."""

    def __init__(self, batch, longest, hidden=4096, ffn=11008, heads=32, kv_heads=8, dim=128,
                 page=64, group=64, dtype=torch.bfloat16, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.batch, self.heads, self.kv_heads, self.dim, self.dtype = batch, heads, kv_heads, dim, dtype

        def weight(n, k):
            w = torch.randn((n, k), generator=g, device="cuda") * k ** -0.5
            return b200k.w4_quantize(w.to(dtype), group=128, zeros=True)

        self.qkv = weight((heads + 2 * kv_heads) * dim, hidden)
        self.out = weight(hidden, heads * dim)
        self.gate_up = weight(2 * ffn, hidden)
        self.down = weight(hidden, ffn)
        self.norms = [(1 + 0.1 * torch.randn(hidden, generator=g, device="cuda")).to(dtype)
                      for _ in range(2)]
        pos = torch.arange(longest, device="cuda")[:, None]
        angle = pos * 10000.0 ** (-torch.arange(0, dim, 2, device="cuda") / dim)
        angle = torch.cat((angle, angle), 1)
        self.cos, self.sin = angle.cos().to(dtype), angle.sin().to(dtype)
        wide = -(-longest // page)
        self.cache = b200k.KVCache4.zeros(batch * wide, page, kv_heads, dim, group)
        # sequence i owns pages in an order of the pool's
        ids = torch.randperm(batch * wide, generator=g, device="cuda")
        self.table = ids.view(batch, wide).int().contiguous()
        self.lengths = torch.zeros(batch, dtype=torch.int32, device="cuda")

    def slots(self, positions):
        """Cache slots of one position per sequence."""
        page = self.cache.page_size
        return self.table.long().gather(1, (positions // page)[:, None])[:, 0] * page + positions % page

    def prompt(self, lengths, seed=1):
        """Fills the cache with random keys and values for each sequence."""
        g = torch.Generator(device="cuda").manual_seed(seed)
        shape = (self.batch, self.kv_heads, self.dim)
        for t in range(int(lengths.max())):
            k = torch.randn(shape, generator=g, device="cuda").to(self.dtype)
            v = torch.randn(shape, generator=g, device="cuda").to(self.dtype)
            here = torch.full((self.batch,), t, device="cuda")
            b200k.kv_cache_write(self.cache, k, v, torch.where(here < lengths, self.slots(here), -1))
        self.lengths.copy_(lengths)

    def step(self, x, residual):
        """One token of every sequence: (stream, block output) from (x, stream)."""
        h, q8, scale = b200k.add_rmsnorm_quant(x, residual, self.norms[0])
        qkv = b200k.w4_matmul(q8, self.qkv, x_scale=scale, out_dtype=self.dtype)
        qkv = qkv.view(self.batch, self.heads + 2 * self.kv_heads, self.dim)
        position = self.lengths.long()
        rotated = self.heads + self.kv_heads
        tables = [t[position].repeat_interleave(rotated, 0) for t in (self.cos, self.sin)]
        qk = b200k.rope(qkv[:, :rotated].reshape(-1, self.dim), *tables)
        qk = qk.view(self.batch, rotated, self.dim)
        b200k.kv_cache_write(self.cache, qk[:, self.heads:], qkv[:, rotated:], self.slots(position))
        self.lengths += 1
        o = b200k.cache_attention(qk[:, None, :self.heads], self.cache, self.table, self.lengths)
        a = b200k.w4_matmul(o.view(self.batch, -1), self.out)
        h, q8, scale = b200k.add_rmsnorm_quant(a, h, self.norms[1])
        gate, up = b200k.w4_matmul(q8, self.gate_up, x_scale=scale, out_dtype=self.dtype).chunk(2, 1)
        return h, b200k.w4_matmul(b200k.swiglu(gate, up), self.down)

    def reference(self, x, residual):
        """step() in float32 from the weights and the cache as they are held; the
        cache must hold the step's own token already (call it after step())."""
        def product(x, w):
            return x @ b200k.w4_matmul(torch.eye(w.k, device="cuda"), w)  # [k, n]

        def norm(h, w):
            return h * w.float() * torch.rsqrt(h.square().mean(1, keepdim=True) + 1e-6)

        h = x.float() + residual.float()
        qkv = product(norm(h, self.norms[0]), self.qkv)
        q = qkv[:, :self.heads * self.dim].view(self.batch, self.heads, self.dim)
        position = self.lengths.long() - 1
        cos, sin = (t.float()[position][:, None] for t in (self.cos, self.sin))
        lo, hi = q.chunk(2, 2)
        q = q * cos + torch.cat((-hi, lo), 2) * sin
        longest = int(self.lengths.max())
        at = torch.arange(longest, device="cuda")
        page = self.cache.page_size
        slots = self.table.long()[:, at // page] * page + at % page
        k, v = (t.float().repeat_interleave(self.heads // self.kv_heads, 2)
                for t in b200k.kv_cache_read(self.cache, slots, dtype=self.dtype))
        z = torch.einsum("bhd,bthd->bht", q, k) * self.dim ** -0.5
        z = z.masked_fill(at >= self.lengths[:, None, None], -float("inf"))
        o = torch.einsum("bht,bthd->bhd", z.softmax(2), v.masked_fill(
            (at >= self.lengths[:, None])[:, :, None, None], 0)).reshape(self.batch, -1)
        h = h + product(o, self.out)
        gate, up = product(norm(h, self.norms[1]), self.gate_up).chunk(2, 1)
        return h, product(torch.nn.functional.silu(gate) * up, self.down)


def relative(a, b):
    return float((a.float() - b.float()).norm() / b.float().norm())


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--batch", type=int, default=16)
    ap.add_argument("--context", type=int, default=1024, help="prompt of the longest sequence")
    ap.add_argument("--steps", type=int, default=16)
    a = ap.parse_args()
    layer = DecoderLayer(a.batch, a.context + a.steps + 2)
    lengths = torch.linspace(a.context // 4, a.context, a.batch, device="cuda").long()
    layer.prompt(lengths)
    x = torch.randn((a.batch, 4096), device="cuda").bfloat16()
    residual = torch.randn((a.batch, 4096), device="cuda").bfloat16()
    layer.step(x, residual)
    h, y = layer.step(x, residual)
    rh, ry = layer.reference(x, residual)
    print(f"one step against float32 from the same weights and cache: stream {relative(h, rh):.4f}, "
          f"block output {relative(y, ry):.4f} (relative)")
    layer.lengths -= 1  # the graph decodes from here
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step(x, residual)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for _ in range(a.steps):
        graph.replay()
    end.record()
    torch.cuda.synchronize()
    print(f"{a.batch} sequences of up to {a.context} tokens, hidden 4096, FFN 11008: "
          f"{start.elapsed_time(end) / a.steps * 1e3:.1f} us per step of one layer")


if __name__ == "__main__":
    main()
