"""Speculative verify steps over an 8-bit paged K/V cache with eviction, on one synthetic attention layer.

A prompt is quantised into the cache; then every step drafts a tree per request (ops.build_trees on random drafter
logits), attends from all its nodes to the cache and to the tree (kv8_attention), accepts a path (ops.accept), adds the
accepted nodes' attention weights to the pages' mass (kv8_page_weights), quantises the accepted keys and values
(kv8_append) and, once a request fills more pages than its budget, drops the least used ones (kv8_evict).

    python examples/kv8_long_context.py [--dtype int8|e4m3] [--steps 8] [--prompt 3000]
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.abspath(os.path.join(os.path.dirname(__file__), "..")))

from mfd_b200 import ops  # noqa: E402
from mfd_b200.kv8_cache import KV8Cache  # noqa: E402


def run(dtype=torch.int8, steps: int = 8, prompt: int = 3000, batch: int = 3, heads: int = 16, kv_heads: int = 4,
        budget: int = 63, modes: int = 4, depth: int = 8, vocab: int = 2048, page: int = 64, keep_pages: int = 40,
        seed: int = 0, log=print) -> dict:
    dev, d = "cuda", 128
    g = torch.Generator(device=dev).manual_seed(seed)
    scale = d ** -0.5

    def weights(*shape):
        return (torch.randn(*shape, generator=g, device=dev) * shape[0] ** -0.5).bfloat16()

    width = heads * d
    embed = torch.randn(vocab, width, generator=g, device=dev).bfloat16()
    wq, wk, wv, head = weights(width, width), weights(width, kv_heads * d), weights(width, kv_heads * d), \
        weights(width, vocab)

    def project(tokens):
        x = embed[tokens]
        b, n = tokens.shape
        return ((x @ wq).view(b, n, heads, d), (x @ wk).view(b, n, kv_heads, d), (x @ wv).view(b, n, kv_heads, d))

    longest = prompt + steps * (depth + 1) + budget
    per_request = -(-longest // page) + 1
    cache = KV8Cache(batch, batch * per_request, kv_heads, per_request, page, d, dtype, dev)
    lens = torch.tensor([prompt - 37 * b for b in range(batch)], dtype=torch.int32, device=dev)
    tokens = torch.randint(0, vocab, (batch, prompt), generator=g, device=dev)
    _, k, v = project(tokens)
    cache.reserve(prompt)
    cache.append(k, v, counts=lens)

    root = tokens[:, -1]
    history = []
    for step in range(steps):
        cache.reserve(depth + 1)
        # drafts: a tree of `budget` nodes behind each request's last token
        logits = torch.randn(batch * modes * depth, vocab, generator=g, device=dev) * 2
        top, ids, _ = ops.topk_logz(logits, budget)
        tree, counts, anc, _ = ops.build_trees(top.view(batch, modes, depth, budget),
                                               ids.view(batch, modes, depth, budget), None, budget)
        nodes = tree[:, 0].clone()
        nodes[:, 0] = root
        q, k, v = project(nodes)
        out, lse = cache.attention(q, scale, k, v, anc, return_lse=True)
        # the target's logits, pulled towards a drafted path so that some of it is accepted
        target = (out.reshape(batch, budget + 1, width) @ head).float()
        child = torch.zeros_like(nodes)
        child.scatter_(1, tree[:, 2].clamp_min(0).flip(1), tree[:, 0].flip(1))
        target.scatter_add_(2, child.unsqueeze(2), torch.full((batch, budget + 1, 1), 20.0, device=dev))
        step_out = ops.accept(target.bfloat16(), nodes, tree[:, 2], max_steps=depth)
        path, commit = step_out["accepted"], step_out["commit_lens"]
        cache.weigh(q, lse, scale, path, commit, decay=0.95)
        cache.append(k, v, path, commit)
        gone = cache.evict(keep_pages)
        root = step_out["bonus"]
        history.append({"committed": commit.tolist(), "evicted": [len(x) for x in gone],
                        "tokens": cache.seq_lens.tolist()})
        log(f"step {step}: committed {history[-1]['committed']}, pages evicted {history[-1]['evicted']}, tokens cached "
            f"{history[-1]['tokens']}")
    if int(cache.status):
        raise RuntimeError("an append found no page")
    return {"history": history, "cache": cache, "out": out}


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--dtype", choices=["int8", "e4m3"], default="int8")
    ap.add_argument("--steps", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=3000)
    a = ap.parse_args()
    run(torch.int8 if a.dtype == "int8" else torch.float8_e4m3fn, a.steps, a.prompt)
