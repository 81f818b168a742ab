"""The attention half of a decoder layer as a server runs it: prompts, then token by token, with the
cache in 4 bits and kept under a budget.

    python examples/decode_layer.py [--steps 40] [--budget 256]

Q4_K projections (fused QKV 5120 -> 10240, O 8192 -> 5120; 64 query heads over 8 key/value heads of
128), rotary positions with three axes (the prompt's second half is an image), the paged 4-bit
cache, attention with accumulated weights, and eviction in place once a sequence is past the budget.
Weights are random; the layer's output is printed as a checksum. Needs a B200.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import busfill_b200 as bf  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM = 5120, 64, 8, 128


def random_q4k(rows, k, gen, dev):
    """Random block_q4_K rows [rows, k / 256 * 144] with small scales."""
    blocks = torch.randint(0, 256, (rows, k // 256, 144), dtype=torch.uint8, generator=gen).to(dev)
    blocks[..., 0:4] = torch.tensor([4e-5, 3e-4], dtype=torch.float16).view(torch.uint8).to(dev)
    return blocks.view(rows, -1)


class Layer:
    def __init__(self, batch, max_tokens, dev="cuda", seed=0):
        gen = torch.Generator().manual_seed(seed)
        self.w_qkv = random_q4k((HEADS + 2 * KV_HEADS) * DIM, HIDDEN, gen, dev)
        self.w_o = random_q4k(HIDDEN, HEADS * DIM, gen, dev)
        self.cos, self.sin = bf.rope_table(4096, DIM, base=1e6, device=dev)
        self.axis = [i * 3 // (DIM // 2) for i in range(DIM // 2)]   # time, height, width
        # pages of every sequence, as many as its longest stay needs
        cols = -(-max_tokens // bf.KV4_PAGE)
        self.pages = bf.kv4_pool(batch * cols, KV_HEADS, DIM, device=dev)
        self.table = torch.arange(batch * cols, dtype=torch.int32, device=dev).view(batch, cols)
        self.kv_len = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.weights = torch.zeros((batch, KV_HEADS, cols * bf.KV4_PAGE), device=dev)

    def __call__(self, x, positions, new):
        """x [tokens, HIDDEN] fp16, the new tokens of the sequences one after another; positions int32
        [3, tokens]; new: tokens of each sequence."""
        dev = x.device
        counts = torch.tensor(new, dtype=torch.int32, device=dev)
        start = torch.nn.functional.pad(counts.cumsum(0, dtype=torch.int32), (1, 0))
        self.kv_len = self.kv_len + counts
        y = torch.nn.functional.rms_norm(x.float(), (HIDDEN,)).half()
        qkv = bf.gemm_q4k(self.w_qkv, y).view(-1, HEADS + 2 * KV_HEADS, DIM)
        q, k = bf.rope_axes(qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV_HEADS], positions, self.cos, self.sin, self.axis)
        bf.kv4_append(self.pages, self.table, self.kv_len, k, qkv[:, HEADS + KV_HEADS:], q_start=start)
        o = bf.attn_kv4(q, self.pages, self.table, self.kv_len, q_start=start, max_q=max(new), weights=self.weights)
        return x + bf.gemm_q4k(self.w_o, o.view(-1, HEADS * DIM))

    def trim(self, budget):
        """Bring every sequence down to `budget` tokens, a quarter of them the latest."""
        _, self.weights, self.kv_len = bf.kv4_evict(self.pages, self.table, self.kv_len, self.weights, budget,
                                                    budget // 4, weights_out=self.weights)


def image_positions(n, dev):
    """Time, height and width of n prompt tokens: text, then an image of the second half."""
    text = n // 2
    i = torch.arange(n, device=dev)
    side = max(1, int((n - text) ** 0.5))
    height, width = text + (i - text) // side, text + (i - text) % side
    return torch.stack([torch.where(i < text, i, text), torch.where(i < text, i, height),
                        torch.where(i < text, i, width)]).int()


def run(steps=40, budget=256, prompts=(300, 170), seed=0):
    dev = torch.device("cuda")
    layer = Layer(len(prompts), max(max(prompts), budget) + steps, dev, seed)
    gen = torch.Generator().manual_seed(seed + 1)
    x = torch.randn((sum(prompts), HIDDEN), generator=gen).half().to(dev)
    y = layer(x, torch.cat([image_positions(n, dev) for n in prompts], 1), list(prompts))
    last = torch.tensor(prompts).cumsum(0) - 1
    x, at = y[last.to(dev)], torch.tensor(prompts, device=dev)
    lengths = []
    for step in range(steps):
        if step % 16 == 0:
            layer.trim(budget)
        x = layer(x, (at + step).expand(3, -1).int().contiguous(), [1] * len(prompts))
        lengths.append(layer.kv_len.tolist())
    if bf.stream_status() != 0:
        raise RuntimeError("a kernel reported a failure")
    return x, lengths, layer


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=40)
    ap.add_argument("--budget", type=int, default=256)
    args = ap.parse_args()
    x, lengths, _ = run(args.steps, args.budget)
    print(f"cached tokens after each step: {lengths}")
    print(f"output: mean {x.float().mean().item():.6f}, rms {x.float().pow(2).mean().sqrt().item():.6f}")


if __name__ == "__main__":
    main()
