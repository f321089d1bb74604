"""One attention layer that keeps its context in the 4-bit cache.

A prompt is taken in chunks (append, then attention over everything before),
then tokens are decoded one at a time: append rotates the new token and writes
it in 4 bits, select picks the blocks that its query reads, attend reads them.
Weights are random, with query heads that look for tokens like their own;
inputs are a text of random subjects, some hundred tokens each, and decoded
tokens return to early ones.  The result is compared with attention over the
unquantised keys and values.

    python examples/kv_decode.py --prompt 20000 --steps 32 --select 64
"""
from __future__ import annotations

import argparse
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "go-fann_b200"))
from gofann.kv_cache import PAGE, KVBatch, KVCache, rope_tables  # noqa: E402


class Layer:
    """Projections, the sequences' caches and their page table."""

    def __init__(self, width: int, heads: int, kv_heads: int, head_dim: int, seqs: int, max_tokens: int,
                 dtype=torch.bfloat16, seed: int = 0):
        g = torch.Generator("cuda").manual_seed(seed)
        self.heads, self.kv_heads, self.d, self.seqs = heads, kv_heads, head_dim, seqs
        normal = lambda *n: torch.randn(*n, generator=g, device="cuda") * width ** -0.5  # noqa: E731
        k = normal(width, kv_heads, 1, head_dim)
        q = 1.5 * (k + 0.5 * normal(width, kv_heads, heads // kv_heads, head_dim))
        self.qkv = torch.cat([x.flatten(1) for x in (q, k, normal(width, kv_heads, head_dim))], 1).to(dtype)
        self.rotary = head_dim // 2  # the other half compares subjects at any distance
        blocks = -(-max_tokens // PAGE)
        self.cache = KVCache.empty(seqs * blocks, kv_heads, head_dim)
        # pages of a real pool are in no order
        self.table = torch.randperm(seqs * blocks, generator=g, device="cuda").int().view(seqs, blocks)
        self.cos, self.sin = rope_tables(max_tokens, self.rotary)
        self.length = 0

    def batch(self, rows: int) -> KVBatch:
        """The next `rows` tokens of every sequence."""
        self.length += rows
        lens = torch.full((self.seqs,), self.length, dtype=torch.int32, device="cuda")
        offset = torch.arange(self.seqs + 1, dtype=torch.int32, device="cuda") * rows
        return KVBatch(self.table, lens, offset, self.seqs * rows, rows)

    def __call__(self, x: torch.Tensor, n_select: int = 0):
        """x [seqs][rows][width] -> out [seqs * rows][heads][head_dim], the
        rotated queries and the unquantised, rotated keys and the values."""
        batch = self.batch(x.shape[1])
        q, k, v = (x.reshape(-1, x.shape[-1]) @ self.qkv).unflatten(-1, (-1, self.d)).split(
            (self.heads, self.kv_heads, self.kv_heads), dim=1)
        q_rot, _, _ = self.cache.append(batch, q, k, v, cos=self.cos, sin=self.sin, rotary_dim=self.rotary)
        ids = self.cache.select(batch, q_rot, n_select=n_select, first=1, recent=2)[0] if n_select else None
        out, _ = self.cache.attend(batch, q_rot, selected=ids)
        return out, q_rot, k, v


def rotated(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    """x [seqs][tokens][heads][d] by the positions 0, 1, .."""
    half = cos.shape[1]
    a, b, rest = x.float().split((half, half, x.shape[-1] - 2 * half), -1)
    c, s = cos[: x.shape[1], None], sin[: x.shape[1], None]
    return torch.cat((a * c - b * s, b * c + a * s, rest), -1)


def run(prompt: int, steps: int, n_select: int, seqs: int = 2, chunk: int = 2048, heads: int = 16, kv_heads: int = 4,
        head_dim: int = 128, width: int = 1024, seed: int = 0):
    """Relative errors of the last decoded token's output against unquantised
    attention over all tokens: (reading all blocks, reading the selected ones),
    and the seconds of a decode step."""
    layer = Layer(width, heads, kv_heads, head_dim, seqs, prompt + steps, seed=seed)
    g = torch.Generator("cuda").manual_seed(seed + 1)
    subjects = torch.randn(seqs, prompt // 150 + 1, width, generator=g, device="cuda")

    def text(first, n):
        at = torch.arange(first, first + n, device="cuda") // 150
        noise = torch.randn(seqs, n, width, generator=g, device="cuda")
        return (0.8 * subjects[:, at % subjects.shape[1]] + 0.6 * noise).to(torch.bfloat16)

    keys, values, at = [], [], 0
    while at < prompt:
        n = min(chunk, prompt - at)
        _, _, k, v = layer(text(at, n))
        keys.append(k.unflatten(0, (seqs, n)).float())
        values.append(v.unflatten(0, (seqs, n)).float())
        at += n
    tokens = [text(151 * i, 1) for i in range(steps)]
    torch.cuda.synchronize()
    start = time.perf_counter()
    for x in tokens:
        out, q, k, v = layer(x, n_select)
        keys.append(k.unflatten(0, (seqs, 1)).float())
        values.append(v.unflatten(0, (seqs, 1)).float())
    torch.cuda.synchronize()
    seconds = (time.perf_counter() - start) / steps

    # the last token again, over all blocks, and in plain torch
    batch = KVBatch(layer.table, torch.full((seqs,), layer.length, dtype=torch.int32, device="cuda"),
                    torch.arange(seqs + 1, dtype=torch.int32, device="cuda"), seqs, 1)
    dense, _ = layer.cache.attend(batch, q)
    batch.check()
    k, v = rotated(torch.cat(keys, 1), layer.cos, layer.sin), torch.cat(values, 1)
    group = heads // kv_heads
    score = torch.einsum("shgd,sthd->shgt", q.float().unflatten(1, (kv_heads, group)), k) * head_dim ** -0.5
    want = torch.einsum("shgt,sthd->shgd", torch.softmax(score, -1), v).flatten(1, 2)
    error = lambda x: float((x.float() - want).norm() / want.norm())  # noqa: E731
    return error(dense), error(out), seconds


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    p.add_argument("--prompt", type=int, default=20000)
    p.add_argument("--steps", type=int, default=32)
    p.add_argument("--select", type=int, default=64, help="blocks of 64 tokens that a decoded token reads; 0 = all")
    p.add_argument("--seqs", type=int, default=2)
    a = p.parse_args()
    dense, sparse, seconds = run(a.prompt, a.steps, a.select, a.seqs)
    print(f"{a.seqs} sequences of {a.prompt} + {a.steps} tokens, {seconds * 1e6:.0f} us a decode step")
    print(f"relative error against unquantised attention: all blocks {dense:.4f}, "
          f"{a.select or 'all'} blocks {sparse:.4f}")


if __name__ == "__main__":
    main()
