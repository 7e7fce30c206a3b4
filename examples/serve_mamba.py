"""Prompts of different lengths, then tokens one by one, through a small stack of Mamba-2, Mamba or linear-attention layers with random weights.

    python examples/serve_mamba.py [--kind mamba2|mamba|attention] [--layers 4] [--batch 8] [--prompt 1000] [--tokens 64]

Every layer call is the package's operators only: INT8 projections behind norms that write codes, short convolution, recurrence,
or linear attention, gated norm; with linear attention every other sequence has a low-rank adapter of its own. The token step of the whole stack is captured once as a CUDA graph."""

import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import linquant_b200  # noqa: E402
from linquant_b200.models import LinearAttentionLayer, Mamba2Layer, MambaLayer  # noqa: E402


def low_rank(N, K, rank=16):
    return torch.randn(rank, K, device="cuda") / K**0.5, torch.randn(N, rank, device="cuda") * 0.1


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--kind", choices=("mamba2", "mamba", "attention"), default="mamba2")
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=1000)
    ap.add_argument("--tokens", type=int, default=64)
    a = ap.parse_args()
    d, dtype = 2560, torch.float16
    if a.kind == "mamba2":
        layers = [Mamba2Layer(d, 80, slots=a.batch, dtype=dtype, seed=i) for i in range(a.layers)]
    elif a.kind == "attention":
        layers = [LinearAttentionLayer(d, 16, slots=a.batch, dtype=dtype, seed=i) for i in range(a.layers)]
        for layer in layers:
            layer.adapt(*([low_rank(*p.codes.shape) for _ in range(a.batch // 2)] or None for p in (layer.in_proj, layer.out_proj)))
    else:
        layers = [MambaLayer(d, 2 * d, slots=a.batch, dtype=dtype, seed=i) for i in range(a.layers)]
    x = torch.randn(a.batch, a.prompt, d, device="cuda", dtype=dtype)
    lengths = torch.randint(1, a.prompt + 1, (a.batch,), device="cuda", dtype=torch.int32)
    slots = torch.arange(a.batch, device="cuda", dtype=torch.int32)
    own = {}  # each sequence's adapter, behind the stack's end: none
    if a.kind == "attention":
        own["adapters"] = torch.where(slots % 2 == 1, slots // 2, a.batch).int()

    def prompt():
        h, r = x, torch.zeros_like(x)
        for layer in layers:
            h, r = layer.prefill(h, r, slots, lengths, **own)
        return h

    if a.kind == "mamba2":  # static scales of the SSD ops, layer by layer
        h, r = x, torch.zeros_like(x)
        for layer in layers:
            layer.calibrate(h, r)
            h, r = layer.prefill(h, r, slots)
    prompt()
    torch.cuda.synchronize()
    t = time.perf_counter()
    h = prompt()
    torch.cuda.synchronize()
    print(f"prompt: {a.batch} x {a.prompt} tokens, {a.layers} layers: {(time.perf_counter() - t) * 1e3:.2f} ms")

    token = h[torch.arange(a.batch, device="cuda"), lengths.long() - 1].clone()

    def step():
        h, r = token, torch.zeros_like(token)
        for layer in layers:
            h, r = layer.step(h, r, slots, **own)
        token.copy_(h)  # what a head and a sampler would choose

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(a.tokens):
        graph.replay()
    torch.cuda.synchronize()
    print(f"tokens: {a.tokens} steps of {a.batch} sequences: {(time.perf_counter() - t) / a.tokens * 1e6:.1f} us a step, {a.layers} layers")
    linquant_b200.check_status()
    assert torch.isfinite(token).all()


if __name__ == "__main__":
    main()
