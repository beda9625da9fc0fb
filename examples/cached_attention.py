"""Attention layers over an 8-bit cache: prompts of several lengths, then tokens one at a time from a replayed HIP graph.

    python examples/cached_attention.py

A step of a layer is linear() (queries, keys and values in one INT8 matrix), rotary(), kv_write(), kv_attention() and linear() again,
in place of the residual stream. kv_plan() gives the step its slots, positions and block tables from the requests' lengths, on the
GPU, so that a decode step reads nothing on the host and is captured once. Weights are random; the program checks that the
tokens fed one at a time get the values that they get all at once.
"""
import sys
from pathlib import Path

import torch

if __name__ == "__main__":
    sys.path.insert(0, str(Path(__file__).resolve().parents[1]))
from wgpkernels_amd import int8 as wq

BLOCK = 16


def int8_weight(n, k, generator):
    """A random (n, k) matrix as INT8 with a scale per channel."""
    w = torch.randn(n, k, generator=generator, device="cuda") * k ** -0.5
    scale = w.abs().amax(1) / 127
    return torch.round(w / scale[:, None]).to(torch.int8), scale


class Layer:
    def __init__(self, width, q_heads, heads, head_dim, pages, generator):
        self.q_heads, self.heads, self.head_dim = q_heads, heads, head_dim
        self.qkv = int8_weight((q_heads + 2 * heads) * head_dim, width, generator)
        self.out = int8_weight(width, q_heads * head_dim, generator)
        self.cache = wq.KVCache(pages, heads, head_dim, BLOCK)

    def step(self, x, plan, tables, turns):
        """x (tokens, width) after this layer, in place."""
        row = wq.linear(x, *self.qkv, mode=path(x), act="rms_norm", eps=1e-6).view(len(x), -1, self.head_dim)
        q, k, v = row.split([self.q_heads, self.heads, self.heads], 1)
        q, k = wq.rotary((q, k), plan.positions, turns)
        wq.kv_write(self.cache, k, v, plan.slots)
        a = wq.kv_attention(q, self.cache, tables, plan.lens, plan.starts)
        return wq.linear(a.flatten(1), *self.out, mode=path(x), residual=x, out=x)


def path(x):
    """Few tokens unquantized, many as INT8 with a remainder: fixed here, so that steps of any size compare; linear() chooses by itself."""
    return "lines" if len(x) <= 4 else "small" if len(x) <= 32 else "exact"


class Model:
    """Layers with a cache each, and the requests' state on the GPU: cached lengths, block tables, the free pages."""

    def __init__(self, requests, most_tokens, layers=2, width=512, q_heads=8, heads=2, head_dim=64, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        each = -(-most_tokens // BLOCK)
        pages = requests * each
        self.layers = [Layer(width, q_heads, heads, head_dim, pages, g) for _ in range(layers)]
        self.turns = wq.rotary_plan((head_dim // 2,), style="halves")
        self.tables = torch.full((requests, each), -1, dtype=torch.int32, device="cuda")
        self.free = torch.randperm(pages, generator=g, device="cuda").int()
        self.past, self.used = torch.zeros(requests, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")

    def step(self, x, new):
        """x: the requests' new tokens (new[r] of request r), one after another; their values after the last layer."""
        plan = wq.kv_plan(self.past, new, self.tables, self.free, self.used, BLOCK, len(x))
        for layer in self.layers:
            layer.step(x, plan, self.tables, self.turns)
        self.past.copy_(plan.lens)
        self.used.copy_(plan.used)
        return x

    def forget(self):
        self.past.zero_()
        self.used.zero_()


def decode_graph(model, x, new):
    """A step of model over the tokens in x, captured; replay() leaves the values in x. The model's requests are forgotten."""
    model.step(x, new)  # kernels loaded and tuned outside the capture
    model.forget()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model.step(x, new)
    model.forget()
    return graph


def run(prompts=(37, 5, 100), tokens=20, seed=1):
    """(values of the last `tokens` tokens of each request fed one at a time, the same fed at once)."""
    requests, g = len(prompts), torch.Generator(device="cuda").manual_seed(seed)
    texts = [torch.randn(n + tokens, 512, generator=g, device="cuda").bfloat16() for n in prompts]
    ints = lambda values: torch.tensor(values, dtype=torch.int32, device="cuda")
    model = Model(requests, max(prompts) + tokens)
    x, one = torch.zeros(requests, 512, dtype=torch.bfloat16, device="cuda"), ints([1] * requests)
    graph = decode_graph(model, x, one)
    model.step(torch.cat([t[:n] for t, n in zip(texts, prompts)]), ints(prompts))
    steps = []
    for i in range(tokens):
        x.copy_(torch.stack([t[n + i] for t, n in zip(texts, prompts)]))
        graph.replay()
        steps.append(x.clone())
    fresh = Model(requests, max(prompts) + tokens)
    whole = fresh.step(torch.cat(texts), ints([n + tokens for n in prompts])).split([n + tokens for n in prompts])
    return torch.stack(steps), torch.stack([w[-tokens:] for w in whole], 1)


if __name__ == "__main__":
    stepwise, at_once = run()
    off = ((stepwise.float() - at_once.float()).norm() / at_once.float().norm()).item()
    print(f"{stepwise.shape[0]} steps of {stepwise.shape[1]} requests: {off:.2%} from the same tokens fed at once")
