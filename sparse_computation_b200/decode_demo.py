"""Decoding with pruned weights: a small decoder stack that runs the products
and the serving operators together.

    python -m sparse_computation_b200.decode_demo --requests 32 --steps 64

Every layer has 80 % magnitude-pruned 512 x 512 q/k/v/o and 2048 x 512 /
512 x 2048 FFN weights (transformer-base shapes, seeded random values).
Activations stay feature-major (512 x requests, fp32) between the products; a
step appends each request's new key and value to a paged cache, rotated by its
position, attends over it, and adds each request's low-rank adapter beside the
q and o projections.  Prints the time of a step.
"""
from __future__ import annotations

import argparse

import torch

from . import CSR, DecodeAttention, LowRankAdapters, PagedKVCache, RotaryTable, SpMMPlan, \
    csr_to_compressed_format_converter
from . import workloads as wl

WIDTH, HEADS, HEAD_DIM, FFN = 512, 8, 64, 2048


def rotation(positions: int, device) -> RotaryTable:
    half = HEAD_DIM // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=device) / half)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq
    return RotaryTable(angle.cos().float(), angle.sin().float())


class Layer:
    def __init__(self, seed: int, requests: int, pages: int, page_size: int, adapters: int, cache_type, device: int = 0):
        def plan(rows, cols, s):
            a = CSR.from_arrays(*wl.magnitude_pruned(rows, cols, 0.80, 0.05, s))
            return SpMMPlan(csr_to_compressed_format_converter(a, 4, 1), requests, device=device)

        self.w = {n: plan(WIDTH, WIDTH, seed + i) for i, n in enumerate("qkvo")}
        self.ffn1, self.ffn2 = plan(FFN, WIDTH, seed + 4), plan(WIDTH, FFN, seed + 5)
        gen = torch.Generator().manual_seed(seed)
        draw = lambda *shape: (torch.randn(*shape, generator=gen) * shape[-1] ** -0.5).to(f"cuda:{device}")
        ranks = [4 + 4 * (i % 4) for i in range(adapters)]
        self.adapters = {n: LowRankAdapters([draw(r, WIDTH) for r in ranks], [draw(WIDTH, r) for r in ranks],
                                            [0.5] * adapters) for n in "qo"}
        self.cache = PagedKVCache.allocate(pages, page_size, HEADS, HEAD_DIM, cache_type, device)
        self.attention = DecodeAttention(self.cache, HEADS, requests)

    def step(self, x, ids, positions, lengths, table, rope):
        rows = lambda y: y.view(HEADS, HEAD_DIM, -1).permute(2, 0, 1)  # feature-major (heads * dim) x requests
        norm = lambda y: y * torch.rsqrt(y.square().mean(0, keepdim=True) + 1e-6)
        h = norm(x)
        q = self.adapters["q"].apply(h, ids, base=self.w["q"].spmm(h))
        q = self.cache.append(rows(self.w["k"].spmm(h)), rows(self.w["v"].spmm(h)), positions, table, rope=rope, q=rows(q))
        mixed = torch.empty_like(h)
        self.attention.attend(q, table, lengths, out=rows(mixed))
        x = self.adapters["o"].apply(mixed, ids, base=x + self.w["o"].spmm(mixed))
        return x + self.ffn2.spmm(torch.relu(self.ffn1.spmm(norm(x))))


def main(argv=None) -> float:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=32)
    ap.add_argument("--steps", type=int, default=64)
    ap.add_argument("--layers", type=int, default=6)
    ap.add_argument("--page", type=int, default=16)
    ap.add_argument("--cache", choices=["f32", "bf16", "f16"], default="bf16")
    a = ap.parse_args(argv)
    kind = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[a.cache]
    each = -(-a.steps // a.page)
    gen = torch.Generator().manual_seed(0)
    layers = [Layer(100 * i, a.requests, a.requests * each, a.page, 8, kind) for i in range(a.layers)]
    table = torch.randperm(a.requests * each, generator=gen).int().view(a.requests, each).cuda()
    ids = torch.randint(-1, 8, (a.requests,), generator=gen).int().cuda()
    rope = rotation(a.steps, table.device)
    x = torch.randn(WIDTH, a.requests, generator=gen).cuda()
    positions = torch.zeros(a.requests, dtype=torch.int32, device="cuda")
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for step in range(a.steps):
        if step == min(3, a.steps - 1):
            begin.record()
        lengths = positions + 1
        for layer in layers:
            x = layer.step(x, ids, positions, lengths, table, rope)
        positions = lengths
    end.record()
    torch.cuda.synchronize()
    for layer in layers:
        layer.cache.check()
        layer.attention.check()
    ms = begin.elapsed_time(end) / (a.steps - min(3, a.steps - 1))
    print(f"{a.requests} requests, {a.layers} layers, {a.cache} cache: {ms:.3f} ms a step, "
          f"{a.requests / ms * 1e3:.0f} tokens/s, |x| {x.norm().item():.4f}")
    return ms


if __name__ == "__main__":
    main()
