"""A decode step as these operators are meant to be used together: a token's row through attention over the 8-bit cache, the experts, the output
matrix and sample(), whose tokens are the next step's, captured in one HIP graph and replayed; against the same steps run eagerly."""
import torch
import pytest

pytestmark = pytest.mark.gpu
WIDTH, HEADS, KV_HEADS, HEAD, VOCABULARY, EXPERTS, HIDDEN, BLOCK = 256, 4, 2, 64, 1000, 8, 96, 16


def int8_weight(g, *shape):
    w = torch.randn(*shape, generator=g, device="cuda") * shape[-1] ** -0.5
    scale = w.abs().amax(-1) / 127
    return torch.round(w / scale[..., None]).to(torch.int8), scale


class Model:
    """Two layers; the branches' sum and the next norm in one call, in place of the residual stream."""

    def __init__(self, wq, requests, most, seed):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.wq, self.requests = wq, requests
        self.embedding = torch.randn(VOCABULARY, WIDTH, generator=g, device="cuda").bfloat16()
        norm = lambda: (1 + 0.1 * torch.randn(WIDTH, generator=g, device="cuda")).bfloat16()
        self.layers = [{"qkv": int8_weight(g, (HEADS + 2 * KV_HEADS) * HEAD, WIDTH), "out": int8_weight(g, WIDTH, HEADS * HEAD), "norms": (norm(), norm()),
                        "router": torch.randn(EXPERTS, WIDTH, generator=g, device="cuda").bfloat16(), "up": int8_weight(g, EXPERTS, 2 * HIDDEN, WIDTH),
                        "down": int8_weight(g, EXPERTS, WIDTH, HIDDEN), "cache": wq.KVCache(requests * -(-most // BLOCK), KV_HEADS, HEAD, BLOCK)}
                       for _ in range(2)]
        self.head, self.last = int8_weight(g, VOCABULARY, WIDTH), norm()
        self.turns = wq.rotary_plan((HEAD // 2,), style="halves")
        self.tables = torch.full((requests, -(-most // BLOCK)), -1, dtype=torch.int32, device="cuda")
        self.free = torch.arange(requests * -(-most // BLOCK), device="cuda").int()
        self.past, self.used = torch.zeros(requests, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
        self.one = torch.ones(requests, dtype=torch.int32, device="cuda")
        self.tokens = torch.arange(requests, device="cuda") * 7
        self.draws = torch.zeros(requests, device="cuda")
        self.options = {"temperature": torch.linspace(0, 1.2, requests, device="cuda"), "top_k": 40, "top_p": 0.9}

    def step(self):
        wq = self.wq
        plan = wq.kv_plan(self.past, self.one, self.tables, self.free, self.used, BLOCK, self.requests)
        stream = self.embedding[self.tokens]
        branch = torch.zeros_like(stream)
        for layer in self.layers:
            prepared, stream = wq.add_prepare(branch, stream, path="small", act_weight=layer["norms"][0], eps=1e-6, out=stream)
            rows = wq.linear_prepared(prepared, *layer["qkv"]).view(self.requests, -1, HEAD)
            q, k, v = rows.split([HEADS, KV_HEADS, KV_HEADS], 1)
            q, k = wq.rotary((q, k), plan.positions, self.turns)
            wq.kv_write(layer["cache"], k, v, plan.slots)
            a = wq.kv_attention(q, layer["cache"], self.tables, plan.lens, plan.starts)
            prepared, stream = wq.add_prepare(wq.linear(a.flatten(1), *layer["out"], mode="small"), stream, path="small", act_weight=layer["norms"][1], eps=1e-6,
                                              out=stream)
            routes = wq.route(prepared.x, layer["router"], 2)
            branch = wq.experts(prepared.x, routes, *layer["up"], *layer["down"])
        prepared, stream = wq.add_prepare(branch, stream, path="block", act_weight=self.last, eps=1e-6, out=stream)
        logits = wq.linear_prepared(prepared, *self.head)
        self.tokens.copy_(wq.sample(logits, self.draws, **self.options))
        self.past.copy_(plan.lens)
        self.used.copy_(plan.used)
        return logits

    def begin(self):
        self.tokens.copy_(torch.arange(self.requests, device="cuda") * 7)
        self.past.zero_()
        self.used.zero_()


def captured(model):
    model.step()
    model.begin()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        logits = model.step()
    model.begin()
    return graph, logits


def test_captured_steps_are_the_eager_ones(wq):
    """Two models' graphs replayed in turn, each beside its own eager steps."""
    steps, draws = 24, torch.rand(24, 5, generator=torch.Generator().manual_seed(0)).cuda()
    models = [Model(wq, requests, steps + 8, seed) for seed, requests in ((1, 5), (2, 1))]
    eager = []
    for model in models:
        captured(model)  # tiles and paths chosen before either way
        model.begin()
        found = []
        for i in range(steps):
            model.draws.copy_(draws[i, :model.requests])
            logits = model.step()
            found.append((logits.clone(), model.tokens.clone()))
        eager.append(found)
    graphs = [captured(model) for model in models]
    for i in range(steps):
        for model, (graph, logits), found in zip(models, graphs, eager):
            model.draws.copy_(draws[i, :model.requests])
            graph.replay()
            assert torch.equal(logits, found[i][0]), f"step {i}"
            assert torch.equal(model.tokens, found[i][1])
            assert model.past.tolist() == [i + 1] * model.requests
    assert len({t for found in eager for _, tokens in found for t in tokens.tolist()}) > 20  # the tokens move
