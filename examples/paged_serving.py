"""Serving with the paged 8-bit cache: prompts, then tokens one at a time.

A toy attention layer (random projections, no trained weights) takes a few
prompts of different lengths, generates tokens for all of them, lets one
finish and another one in, and compares every output with attention computed
plainly from the unquantised keys and values.

    python examples/paged_serving.py [--codes int8|e4m3]
"""
from __future__ import annotations

import argparse
import importlib
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
serving = importlib.import_module("cupilot-kernels_b200.serving")

HEADS, KV_HEADS, DIM, WIDTH = 8, 2, 64, 256


def plain(q, k, v, causal):
    """softmax(q k^T / sqrt(dim)) v in fp32: q (n, heads, dim), k and v (m, kv_heads, dim)."""
    k, v = (x.float().repeat_interleave(HEADS // KV_HEADS, 1) for x in (k, v))
    z = torch.einsum("nhd,mhd->hnm", q.float(), k) / math.sqrt(DIM)
    if causal:
        z = z.masked_fill(torch.ones(z.shape[1:], dtype=torch.bool, device=z.device).triu(1), -math.inf)
    return torch.einsum("hnm,mhd->nhd", z.softmax(-1), v)


def main(codes="int8", prompts=(37, 5, 130), steps=20, seed=0):
    """Runs the example; returns the largest relative error of the prompts' and the tokens' outputs."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    weight = torch.randn(WIDTH, (HEADS + 2 * KV_HEADS) * DIM, generator=g, device="cuda").bfloat16() / WIDTH ** 0.5
    cache = serving.PagedCache(layers=1, requests=len(prompts), max_tokens=256, blocks=64,
                               kv_heads=KV_HEADS, dim=DIM, codes=codes)
    kept = [[] for _ in prompts]             # each request's (k, v), to compare with
    worst = {"prompt": 0.0, "token": 0.0}

    def project(n):
        x = torch.randn(n, WIDTH, generator=g, device="cuda").bfloat16()
        qkv = (x @ weight).view(n, HEADS + 2 * KV_HEADS, DIM)
        return qkv[:, :HEADS], qkv[:, HEADS:HEADS + KV_HEADS], qkv[:, HEADS + KV_HEADS:]

    def run(new_lens, kind):
        cache.begin(new_lens)
        q, k, v = project(sum(new_lens))
        out = cache.prefill(0, q, k, v) if kind == "prompt" else cache.decode(0, q, k, v)
        at = 0
        for r, n in enumerate(new_lens):
            if n == 0:
                continue
            kept[r].append((k[at:at + n], v[at:at + n]))
            want = plain(q[at:at + n], torch.cat([x for x, _ in kept[r]]), torch.cat([x for _, x in kept[r]]),
                         kind == "prompt")
            worst[kind] = max(worst[kind], ((out[at:at + n].float() - want).norm() / want.norm()).item())
            at += n

    run(list(prompts), "prompt")
    for _ in range(steps):
        run([1] * len(prompts), "token")
    # One request ends; another takes its row while the rest wait, then all go on.
    cache.release(0)
    kept[0] = []
    run([50] + [0] * (len(prompts) - 1), "prompt")
    run([0] + [1] * (len(prompts) - 1), "token")
    for _ in range(steps):
        run([1] * len(prompts), "token")
    return worst


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--codes", choices=sorted(serving.CODES), default="int8")
    for kind, err in main(ap.parse_args().codes).items():
        print(f"{kind}: largest relative error {err:.2e}")
