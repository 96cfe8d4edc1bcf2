"""A small server loop over a K/V cache in pages: prompts read in chunks beside
sequences in generation, one append_paged() and one attend_paged() per layer and
step, checked against rope() and prefill() on whole contiguous sequences.

    python flash-attention-cuda_b200/paged_serving.py [--steps 24] [--chunk 96]

The layer is an attention block with random weights; a step's "next token" is
its normalised output row, so that generation depends on what the cache holds.
"""

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))

import torch  # noqa: E402

import flashattn_cuda as fa  # noqa: E402


class Block:
    """q, k, v and output projections of one attention layer."""

    def __init__(self, heads, kv_heads, dim, dtype):
        self.heads, self.kv_heads, self.dim = heads, kv_heads, dim
        width = heads * dim
        self.qkv = (torch.randn(width, (heads + 2 * kv_heads) * dim, device="cuda")
                    * width ** -0.5).to(dtype)
        self.out = (torch.randn(width, width, device="cuda") * width ** -0.5).to(dtype)
        self.freqs, self.amplitude = fa.rope_frequencies(dim, scaling="linear", factor=2.0)

    def project(self, x):
        qkv = (x @ self.qkv).unflatten(-1, (self.heads + 2 * self.kv_heads, self.dim))
        return qkv.split((self.heads, self.kv_heads, self.kv_heads), dim=-2)

    def finish(self, o):
        y = o.flatten(-2) @ self.out
        return torch.nn.functional.normalize(y.float(), dim=-1).to(y.dtype) * y.shape[-1] ** 0.5


class Pages:
    """A pool of pages and which of them each request has."""

    def __init__(self, block, pages, rows, requests, dtype):
        size = (pages, block.kv_heads, rows, block.dim)
        self.k = torch.empty(size, device="cuda", dtype=dtype)
        self.v = torch.empty(size, device="cuda", dtype=dtype)
        self.rows, self.free = rows, list(range(pages))
        self.table = torch.full((requests, pages), -1, dtype=torch.int32)
        self.held = [0] * requests

    def grow(self, request, length):
        while self.held[request] * self.rows < length:
            self.table[request, self.held[request]] = self.free.pop()
            self.held[request] += 1


def serve(block, prompts, steps, chunk, page_rows, dtype):
    """Feeds every prompt in chunks, then its own outputs; returns all inputs
    and outputs of each request, in order."""
    n = len(prompts)
    total = sum(len(p) + steps for p in prompts)
    pages = Pages(block, total // page_rows + n, page_rows, n, dtype)
    inputs = [list(p) for p in prompts]
    outputs = [[] for _ in prompts]
    while any(len(o) < len(p) + steps for o, p in zip(outputs, prompts)):
        # every request brings what it has: a chunk of its prompt, one
        # generated token, or nothing when it is done
        news = []
        for r in range(n):
            left = len(prompts[r]) + steps - len(outputs[r])
            news.append(min(len(inputs[r]) - len(outputs[r]), chunk, left))
            pages.grow(r, len(outputs[r]) + news[r])
        x = torch.stack([inputs[r][len(outputs[r]) + i] for r in range(n) for i in range(news[r])])
        starts = torch.tensor([0] + news).cumsum(0).to(torch.int32).cuda()
        lens = torch.tensor([len(outputs[r]) + news[r] for r in range(n)], dtype=torch.int32).cuda()
        table = pages.table.cuda()
        q, k, v = block.project(x)
        q = fa.append_paged(k, v, starts, pages.k, pages.v, table, lens, q=q, freqs=block.freqs,
                            amplitude=block.amplitude)
        o = fa.attend_paged(q, starts, pages.k, pages.v, table, lens, block.dim ** -0.5)
        y, at = block.finish(o), 0
        for r in range(n):
            outputs[r].extend(y[at:at + news[r]])
            at += news[r]
            if len(outputs[r]) >= len(inputs[r]):
                inputs[r].append(outputs[r][-1])
    return inputs, outputs


def whole(block, x):
    """The same layer on a whole contiguous sequence."""
    q, k, v = (t.transpose(0, 1)[None] for t in block.project(x))
    positions = torch.arange(x.shape[0], device="cuda", dtype=torch.int32)
    q, k = fa.rope(q, k, positions, block.freqs, amplitude=block.amplitude)
    o = fa.prefill(q, k, v.contiguous(), True, block.dim ** -0.5)
    return block.finish(o[0].transpose(0, 1))


def main(steps=24, chunk=96, page_rows=16, heads=14, kv_heads=2, dim=64, seed=0):
    torch.manual_seed(seed)
    dtype = torch.bfloat16
    block = Block(heads, kv_heads, dim, dtype)
    prompts = [torch.randn(n, heads * dim, device="cuda").to(dtype) for n in (5, 333, 64, 1)]
    inputs, outputs = serve(block, prompts, steps, chunk, page_rows, dtype)
    worst = 0.0
    for x, y in zip(inputs, outputs):
        got, want = torch.stack(y).float(), whole(block, torch.stack(x[:len(y)])).float()
        worst = max(worst, ((got - want).norm() / want.norm()).item())
    assert fa.take_device_error() == 0
    print(f"{len(prompts)} requests, {sum(map(len, outputs))} tokens in pages of {page_rows} rows: "
          f"relative difference from whole sequences {worst:.2e}")
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=24)
    ap.add_argument("--chunk", type=int, default=96)
    ap.add_argument("--page-rows", type=int, default=16)
    args = ap.parse_args()
    main(args.steps, args.chunk, args.page_rows)
