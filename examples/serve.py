"""Serving a small decoder with the paged key-value cache operators.

    python examples/serve.py [--steps N] [--layers L]

A few requests of different lengths arrive.  Their prompts are read in one
packed pass per layer (kv_append rotates queries and keys by position and
fills the cache, prompt_attention attends), then tokens are decoded greedily
for all requests at once, one step a time (kv_append of the new token, then
paged_decode over the cache), with the step captured in a CUDA graph.  At the end
every request is computed again from its whole text, without a cache and in
32 bits, and the last logits are compared.  Weights are random.
"""

import argparse
import math
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ktir_cpu_b200 import (check_status, kv_append, paged_decode, prompt_attention,  # noqa: E402
                           rotary_table)

VOCAB, HEADS, KV_HEADS, DIM, WIDTH, PAGE = 512, 8, 2, 64, 256, 16


class Layer:
    def __init__(self, gen, device):
        rand = lambda *s: (torch.randn(*s, generator=gen, device=device) / math.sqrt(s[0])).bfloat16()  # noqa: E731
        self.qkv = rand(WIDTH, (HEADS + 2 * KV_HEADS) * DIM)
        self.out = rand(HEADS * DIM, WIDTH)
        self.up, self.down = rand(WIDTH, 2 * WIDTH), rand(2 * WIDTH, WIDTH)


class Cache:
    """Pages of every layer, handed out as requests grow."""

    def __init__(self, layers, pages, device):
        shape = (pages, PAGE, KV_HEADS, DIM)
        self.k = [torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(layers)]
        self.v = [torch.zeros(shape, dtype=torch.bfloat16, device=device) for _ in range(layers)]
        self.free = list(range(pages))[::-1]

    def take(self, n):
        return [self.free.pop() for _ in range(n)]


def norm(x):
    x = x.float()
    return (x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6)).bfloat16()


def forward(layers, embedding, tokens, attend):
    """Logits of `tokens` [n]; attend(layer index, q, k, v) -> [n, heads, dim]."""
    x = embedding[tokens]
    for i, layer in enumerate(layers):
        qkv = (norm(x) @ layer.qkv).view(len(tokens), -1, DIM)
        q, k, v = qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:]
        x = x + attend(i, q, k, v).flatten(1) @ layer.out
        x = x + torch.relu(norm(x) @ layer.up) @ layer.down
    return norm(x) @ embedding.t()


def whole_text(layers, embedding, tokens, table):
    """The last token's logits without a cache, attention in 32 bits."""
    n = len(tokens)

    def attend(i, q, k, v):
        c, s = table[:n, None, :DIM // 2], table[:n, None, DIM // 2:]
        turn = lambda a, b: torch.cat([a * c - b * s, b * c + a * s], -1).bfloat16().float()  # noqa: E731
        q, k = (turn(*t.float().chunk(2, -1)) for t in (q, k))
        k, v = (t.float().repeat_interleave(HEADS // KV_HEADS, 1) for t in (k, v))
        x = torch.einsum("nhd,mhd->hnm", q, k) * DIM ** -0.5
        x = x.masked_fill(torch.ones(n, n, dtype=torch.bool, device=x.device).triu(1), -math.inf)
        return torch.einsum("hnm,mhd->nhd", x.softmax(-1), v).bfloat16()

    return forward(layers, embedding, tokens, attend)[-1]


def main(steps=32, n_layers=2, prompts=(37, 5, 120, 64, 1), seed=0):
    if steps < 1 or min(prompts) < 1:
        raise ValueError("needs at least one step, and prompts of at least one token")
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    layers = [Layer(gen, device) for _ in range(n_layers)]
    embedding = (torch.randn(VOCAB, WIDTH, generator=gen, device=device) / math.sqrt(WIDTH)).bfloat16()
    table = rotary_table(max(prompts) + steps + 1, DIM, device=device)
    texts = [torch.randint(0, VOCAB, (n,), generator=gen, device=device).tolist() for n in prompts]
    index = lambda x: torch.tensor(x, dtype=torch.int32, device=device)  # noqa: E731

    # pages for the whole of every request
    need = [-(-(n + steps) // PAGE) for n in prompts]
    cache = Cache(n_layers, sum(need), device)
    rows = [cache.take(n) for n in need]
    pages = index([r + [0] * (max(need) - len(r)) for r in rows])

    # -- the prompts, packed ---------------------------------------------------------
    offsets = index([sum(prompts[:i]) for i in range(len(prompts) + 1)])
    positions = index([p for n in prompts for p in range(n)])
    slots = index([rows[b][p // PAGE] * PAGE + p % PAGE for b, n in enumerate(prompts) for p in range(n)])

    def read(i, q, k, v):
        at = slots.long()
        q = kv_append(k, v, cache.k[i], cache.v[i], slots, q=q, positions=positions, table=table)
        turned = cache.k[i][at // PAGE, at % PAGE]          # the rotated keys, in the order of the prompts
        return prompt_attention(q, turned, v, offsets)

    logits = forward(layers, embedding, torch.tensor(sum(texts, []), device=device), read)
    new = logits[offsets[1:].long() - 1].argmax(-1)

    # -- one token per request and step, captured once ----------------------------------
    lengths, position = index(prompts), index(prompts)      # keys so far; the new token's position

    def step():
        at = pages.gather(1, (position // PAGE).long()[:, None])[:, 0] * PAGE + position % PAGE
        lengths.copy_(position + 1)

        def attend(i, q, k, v):
            q = kv_append(k, v, cache.k[i], cache.v[i], at, q=q, positions=position, table=table)
            return paged_decode(q, cache.k[i], cache.v[i], pages, lengths)

        out = forward(layers, embedding, new, attend)
        new.copy_(out.argmax(-1))
        position.add_(1)
        return out

    history, last = [new.clone()], logits[offsets[1:].long() - 1]
    if steps > 1:
        step()                                               # once outside the graph; its token is
        new.copy_(history[0])                                # decoded again, and written again
        position.copy_(index(prompts))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            last = step()
        for _ in range(steps - 1):
            graph.replay()
            history.append(new.clone())
    for tokens in history:
        for b, t in enumerate(tokens.tolist()):
            texts[b].append(t)
    check_status()

    # -- against the whole texts, without their last tokens --------------------------------
    worst = 0.0
    for b, text in enumerate(texts):
        want = whole_text(layers, embedding, torch.tensor(text[:-1], device=device), table).float()
        worst = max(worst, float((last[b].float() - want).abs().max() / want.abs().max()))
    print(f"{len(texts)} requests, prompts of {list(prompts)} tokens, {steps} tokens decoded each; "
          f"last logits within {worst:.4f} of the whole text without a cache")
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--layers", type=int, default=2)
    a = ap.parse_args()
    main(a.steps, a.layers)
