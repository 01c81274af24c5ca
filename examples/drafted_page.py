"""One attention layer reading a page with a 4-bit cache of a bounded window, its tokens drafted as trees.

    python examples/drafted_page.py [rows of the prompt] [steps]

The cache operators together, as a decoder with a draft model would use them (libocrcuda.so has to be built, a GPU is
needed):

  op_kv_write          the prompt's keys and values, a chunk of rows at a time, quantised to q4_0 into a ring cache that
                       holds the first four positions and the last 512, however long the page grows
  op_attention_window  the chunk's rows attend what the cache holds
  op_kv_write, op_attention_tree
                       each step: a tree of drafted tokens is written behind the committed rows, all drafts attend at once
  op_kv_keep           the rows of the accepted path (here: the path to the draft that a rule picks) move together, and
                       the next step goes on behind them

At the end the accepted tokens are read again one at a time, the plain way, into a second cache: every output has to be
that of the drafts.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "historic-htr-ocr_b200"))
import ocr_b200 as ocr  # noqa: E402

DIM, HEADS, KV, D = 1024, 16, 8, 128  # the text decoder's widths
WINDOW, SINKS, CHUNK, DRAFTS = 512, 4, 128, 12
SCALE = 1 / math.sqrt(D)


def ring_cache() -> ocr.KvCache:
    n_rows = SINKS + WINDOW + CHUNK  # (a call's rows may not push out what its first row sees)
    q = [torch.zeros(1, KV, n_rows, D // 2, dtype=torch.uint8, device="cuda") for _ in "kv"]
    s = [torch.zeros(1, KV, n_rows, D // 32, dtype=torch.float16, device="cuda") for _ in "kv"]
    return ocr.KvCache("q4_0", *q, *s, d_head=D, window=WINDOW, sinks=SINKS, ring=True)


class Layer:
    """q, k, v of token embeddings at given positions: a projection, a norm per head, the rotary turn"""

    def __init__(self, seed: int):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.w = torch.randn(DIM, (HEADS + 2 * KV) * D, device="cuda", generator=g) / math.sqrt(DIM)
        self.freq = 1e6 ** (-torch.arange(D // 2, device="cuda") / (D // 2))

    def __call__(self, x: torch.Tensor, positions: torch.Tensor):
        y = (x @ self.w).view(1, -1, HEADS + 2 * KV, D)
        qk = y[:, :, :HEADS + KV]
        qk = qk / qk.square().mean(-1, keepdim=True).sqrt()
        a = (positions[:, None].float() * self.freq)[None, :, None]
        lo, hi = qk[..., :D // 2], qk[..., D // 2:]
        qk = torch.cat([lo * a.cos() - hi * a.sin(), hi * a.cos() + lo * a.sin()], -1)
        return qk[:, :, :HEADS], qk[:, :, HEADS:], y[:, :, HEADS + KV:].contiguous()


def tree(g: torch.Generator) -> list[int]:
    """parents: each draft follows one of the four before it, or the last committed token"""
    return [-1] + [int(torch.randint(max(-1, i - 4), i, (), generator=g)) for i in range(1, DRAFTS)]


def main(prompt: int = 1500, steps: int = 20) -> float:
    """→ the largest difference between a draft's output and the plain way's, relative to the largest output"""
    ctx = ocr.Context(0)
    stream = torch.cuda.ExternalStream(ctx.stream())
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):  # everything on the context's stream: the operators queue in order with torch's work
        layer, cache = Layer(1), ring_cache()
        g, gd = torch.Generator().manual_seed(2), torch.Generator(device="cuda").manual_seed(3)
        page = torch.randn(prompt, DIM, device="cuda", generator=gd)
        for a in range(0, prompt, CHUNK):
            rows = page[a:a + CHUNK]
            q, k, v = layer(rows, torch.arange(a, a + len(rows), device="cuda"))
            out, pos = torch.empty_like(q), torch.tensor([a], dtype=torch.int32, device="cuda")
            ocr.op_kv_write(ctx, cache, k, v, pos)
            ocr.op_attention_window(ctx, cache, q.contiguous(), out, pos, SCALE)
        done, kept_x, kept_out = prompt, [], []
        for _ in range(steps):
            parent = tree(g)
            depth = []
            for p in parent:
                depth.append(0 if p < 0 else depth[p] + 1)
            x = torch.randn(DRAFTS, DIM, device="cuda", generator=gd)
            q, k, v = layer(x, done + torch.tensor(depth, device="cuda"))
            out = torch.empty_like(q)
            pos = torch.tensor([done], dtype=torch.int32, device="cuda")
            ocr.op_kv_write(ctx, cache, k, v, pos)
            ocr.op_attention_tree(ctx, cache, q.contiguous(), out, pos,
                                  torch.tensor([parent], dtype=torch.int32, device="cuda"), SCALE)
            # a rule in the place of the model's judgement: the longest path's end
            path, i = [], max(range(DRAFTS), key=lambda j: depth[j])
            while i >= 0:
                path.append(i)
                i = parent[i]
            path.reverse()
            ocr.op_kv_keep(ctx, [cache], pos, torch.tensor([path + [0] * (DRAFTS - len(path))], dtype=torch.int32, device="cuda"),
                           torch.tensor([len(path)], dtype=torch.int32, device="cuda"))
            kept_x.append(x[path])
            kept_out.append(out[0, path])
            done += len(path)
        # the plain way: the same tokens, one at a time
        cache, tokens = ring_cache(), torch.cat([page] + kept_x)
        worst = 0.0
        drafted = torch.cat(kept_out)
        for a in list(range(0, prompt, CHUNK)) + list(range(prompt, done)):
            rows = tokens[a:min(a + CHUNK, prompt)] if a < prompt else tokens[a:a + 1]
            q, k, v = layer(rows, torch.arange(a, a + len(rows), device="cuda"))
            out, pos = torch.empty_like(q), torch.tensor([a], dtype=torch.int32, device="cuda")
            ocr.op_kv_write(ctx, cache, k, v, pos)
            ocr.op_attention_window(ctx, cache, q.contiguous(), out, pos, SCALE)
            if a >= prompt:
                worst = max(worst, float((out[0, 0] - drafted[a - prompt]).abs().max() / drafted.abs().max()))
        ctx.sync()
    held = sum(cache.nbytes()) * 2
    print(f"{done - prompt} tokens accepted in {steps} steps of {DRAFTS} drafts; {held / 1024:.0f} KB of cache for "
          f"{done} positions; drafts and plain steps differ by {worst:.1e} of the largest output")
    return worst


if __name__ == "__main__":
    main(*map(int, sys.argv[1:3]))
