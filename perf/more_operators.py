"""Workloads of a decode step between its attention and its next token, around the INT8 linears.

Kinds of case ("op"):
- "add":     the residual's addition, RMS norm of the sum, and the sum prepared for an INT8 linear's path ("path"): what the
             8-bit codes stand for comes back, beside the sum;
- "experts": a whole mixture-of-experts layer of INT8 weights for a few tokens: the router's product, its choice, and the
             chosen experts' gated feed-forward blocks, weighted and added (to a residual);
- "sample":  a token of every row of logits by given random numbers, with temperature, top-k, top-p and min-p.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
DEVICE = "cuda"
EPS = 1e-6


def add_case(tokens, k, path, dtype="bf16", rotation=0, scaled=False, weight=True):
    return {"op": "add", "tokens": tokens, "k": k, "path": path, "dtype": dtype, "rotation": rotation, "scaled": scaled, "weight": weight}


def experts_case(tokens, k, hidden, experts, top, dtype="bf16", score="softmax", biased=False, normalise=True, factor=1.0, residual=False):
    return {"op": "experts", "tokens": tokens, "k": k, "hidden": hidden, "experts": experts, "top": top, "dtype": dtype, "score": score,
            "biased": biased, "normalise": normalise, "factor": factor, "residual": residual}


def sample_case(rows, vocabulary, dtype="bf16", mixed=False, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    return {"op": "sample", "rows": rows, "vocabulary": vocabulary, "dtype": dtype, "mixed": mixed, "temperature": temperature, "top_k": top_k,
            "top_p": top_p, "min_p": min_p}


def listed():
    return [
        # one user's decode step, unquantized activations for the few-token linears: all latency
        {"name": "add_token_1", **add_case(1, 5120, "small")},
        # batched decode: one scale a token (W8A8), the branch scaled per channel
        {"name": "add_decode_32", **add_case(32, 5120, "row", dtype="fp16", scaled=True)},
        # a ragged text context in full precision (codes and their remainder), a last block of 8 channels
        {"name": "add_context_333", **add_case(333, 4104, "exact", dtype="fp16")},
        # a whole video latent for the block path
        {"name": "add_latent_32760", **add_case(32760, 5120, "block", scaled=True)},
        # one user's decode step: eight experts of 64
        {"name": "experts_token_1", **experts_case(1, 2048, 1024, 64, 8, residual=True)},
        # a handful of tokens, odd sizes, logistic scores with a correction bias for the choice
        {"name": "experts_ragged_5", **experts_case(5, 1552, 592, 21, 3, dtype="fp16", score="sigmoid", biased=True, factor=2.5)},
        # batched decode over many small experts: nearly all of them are read
        {"name": "experts_decode_32", **experts_case(32, 2048, 768, 128, 8, residual=True)},
        # few large experts, many tokens each
        {"name": "experts_wide_100", **experts_case(100, 5120, 1536, 16, 4, dtype="fp16")},
        # one user's next token: FP32 logits, the usual truncations
        {"name": "sample_token_1", **sample_case(1, 131072, dtype="fp32", temperature=0.7, top_k=50, top_p=0.9)},
        # a batch whose requests each bring their own parameters, some of them greedy
        {"name": "sample_mixed_64", **sample_case(64, 131072, mixed=True)},
        # a larger batch over an odd vocabulary, no truncation but a floor
        {"name": "sample_plain_200", **sample_case(200, 50001, dtype="fp16", min_p=0.02)},
    ]


def _log(rng, low, high):
    """An integer whose logarithm is uniform over [low, high]."""
    return max(low, min(high, round(low * (high / low) ** rng.random())))


def draw(rng):
    op = rng.choice(["add", "experts", "experts", "sample"])
    if op == "add":
        k = rng.choice([512, 1024, 1536, 2056, 4104, 5120, 8192, 8200, 13824])
        rotation = rng.choice([0, 0, 16, 64, 256])
        path = rng.choice(["small", "block", "exact", "row"])
        return add_case(_log(rng, 1, 32760 * 4096 // k), k, path, rng.choice(["bf16", "fp16"]), rotation if rotation and k % rotation == 0 else 0,
                        rng.random() < 0.5, rng.random() < 0.8)
    if op == "experts":
        while True:
            experts = _log(rng, 2, 160)
            c = experts_case(_log(rng, 1, 128), 16 * rng.randint(16, 320), 16 * rng.randint(8, 128), experts, rng.randint(1, min(8, experts)),
                             rng.choice(["bf16", "fp16"]), rng.choice(["softmax", "sigmoid"]), rng.random() < 0.3, rng.random() < 0.7,
                             rng.choice([1.0, 2.5]), rng.random() < 0.5)
            if 3 * experts * c["k"] * c["hidden"] <= 6e8:
                return c
    vocabulary = _log(rng, 1000, 262144)
    most = min(256, 64 * 131072 // vocabulary)
    if rng.random() < 0.5:
        return sample_case(_log(rng, 1, most), vocabulary, rng.choice(["bf16", "fp16", "fp32"]), mixed=True)
    return sample_case(_log(rng, 1, most), vocabulary, rng.choice(["bf16", "fp16", "fp32"]), False, round(rng.uniform(0.4, 1.5), 2),
                       rng.choice([0, 1, 40, 1000]), rng.choice([1.0, 0.95, 0.5]), rng.choice([0.0, 0.1]))


def work(case):
    c = case
    if c["op"] == "add":
        # the branch and the residual in, the sum and the values out; between them the codes, written and read
        codes = {"small": 0, "block": 1, "row": 1, "exact": 2}[c["path"]]
        values = c["tokens"] * c["k"]
        return {"bytes": values * (6 + (2 + 2 * codes if codes else 2)), "flops": 8 * values}
    if c["op"] == "experts":
        chosen = c["experts"] * (1 - (1 - c["top"] / c["experts"]) ** c["tokens"])  # of tokens that choose independently
        weights = 3 * c["k"] * c["hidden"]
        rows = c["tokens"] * c["k"]
        return {"bytes": int(chosen * (weights + 4 * (2 * c["hidden"] + c["k"]))) + 2 * c["experts"] * c["k"] + 2 * rows * (3 if c["residual"] else 2)
                + 8 * c["tokens"] * c["top"], "flops": 2 * c["tokens"] * (c["top"] * weights + c["experts"] * c["k"])}
    size = 4 if c["dtype"] == "fp32" else 2
    return {"bytes": c["rows"] * (c["vocabulary"] * size + 12), "flops": 4 * c["rows"] * c["vocabulary"]}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _inputs(c, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device=DEVICE)
    uniform = lambda *shape: torch.rand(*shape, generator=g, device=DEVICE)
    s, d = {"case": c}, DTYPES[c["dtype"]]
    if c["op"] == "add":
        # a residual stream: some channels far larger than the others
        gain = torch.where(uniform(c["k"]) < 0.01, 20.0, 1.0)
        s["x"], s["residual"] = normal(c["tokens"], c["k"]).to(d), normal(c["tokens"], c["k"]).mul_(2 * gain).to(d)
        s["scale"] = (0.3 + 0.2 * normal(c["k"])).to(d) if c["scaled"] else None
        s["weight"] = (1 + 0.2 * normal(c["k"])).to(d) if c["weight"] else None
        return s
    if c["op"] == "experts":
        t, k, f, e = c["tokens"], c["k"], c["hidden"], c["experts"]
        # normed rows with a common part, which the router prefers for some experts: these get more tokens
        common = normal(k)
        x = normal(t, k) + 0.5 * common
        s["x"] = (x / x.square().mean(1, keepdim=True).sqrt()).to(d)
        s["router"] = ((normal(e, k) + 0.02 * normal(e, 1) * common) * 1.5 * k ** -0.5).to(d)
        s["bias"] = 0.05 * normal(e) if c["biased"] else None
        for name, rows, width in (("gate_up", 2 * f, k), ("down", k, f)):
            codes = torch.empty(e, rows, width, dtype=torch.int8, device=DEVICE)
            step = max(1, (1 << 27) // (rows * width))
            for at in range(0, e, step):
                codes[at:at + step] = normal(min(step, e - at), rows, width).mul_(35).round_().clamp_(-127, 127)
            s[name], s[name + "_scale"] = codes, (0.6 + 0.8 * uniform(e, rows)) / 35 * width ** -0.5
        s["residual"] = (2 * normal(t, k)).to(d) if c["residual"] else None
        return s
    n, v = c["rows"], c["vocabulary"]
    logits = normal(n, v).mul_(2.0)
    # a few hundred likely tokens a row, from certain to undecided
    likely = min(300, v)
    at = torch.randint(0, v, (n, likely), generator=g, device=DEVICE)
    logits.scatter_add_(1, at, -torch.log(uniform(n, likely).clamp_(min=1e-6)) * (0.5 + 3 * uniform(n, 1)))
    s["logits"] = logits.to(d)
    s["draws"] = uniform(n)
    if c["mixed"]:
        pick = lambda values, dtype: torch.tensor(values, dtype=dtype, device=DEVICE)[torch.randint(0, len(values), (n,), generator=g, device=DEVICE)]
        s["options"] = {"temperature": pick([0.0, 0.6, 0.8, 1.0, 1.0, 1.3], torch.float32), "top_k": pick([0, 0, 1, 20, 50, 1000], torch.int32),
                        "top_p": pick([1.0, 1.0, 0.95, 0.8, 0.3], torch.float32), "min_p": pick([0.0, 0.0, 0.0, 0.05], torch.float32)}
    else:
        s["options"] = {name: c[name] for name in ("temperature", "top_k", "top_p", "min_p")}
    return s


def prepare(case, seed):
    return _inputs({k: v for k, v in case.items() if k != "name"}, seed)


# ---- plain forms ----------------------------------------------------------------------------------------------------
def _rotation(group):
    """The orthogonal matrix of a group: along every base-4 digit of the place, the four values' sum less twice the opposite one."""
    step = (1 - 2 * torch.eye(4, dtype=torch.float64).flip(0)) / 2
    whole = step
    while len(whole) < group:
        whole = torch.kron(step, whole)
    return whole.to(DEVICE)


def _add_plain(s):
    c, d = s["case"], s["x"].dtype
    branch = s["x"].float() if s["scale"] is None else s["x"].float() * s["scale"].float()
    total = (s["residual"].float() + branch).to(d)
    v = total.float()
    v = v / (v.square().mean(1, keepdim=True) + EPS).sqrt()
    if s["weight"] is not None:
        v = v * s["weight"].float()
    if c["rotation"]:
        v = (v.view(-1, c["rotation"]) @ _rotation(c["rotation"]).float()).view(v.shape)
    if c["path"] != "small":
        blocks = torch.nn.functional.pad(v, (0, -c["k"] % 128)).unflatten(1, (-1, 128)) if c["path"] == "block" else v
        step = blocks.abs().amax(-1, keepdim=True) / 127
        parts = blocks / torch.where(step > 0, step, 1.0)
        codes = parts.round()
        if c["path"] == "exact":
            codes = codes + ((parts - codes) * 254).round() / 254
        v = (codes * step).reshape(len(v), -1)[:, :c["k"]]
    return {"sum": total, "values": v.to(d)}


def _route_plain(s):
    c = s["case"]
    logits = s["x"].double() @ s["router"].double().T
    scores = torch.exp(logits - logits.amax(1, keepdim=True)) if c["score"] == "softmax" else 1 / (1 + torch.exp(-logits))
    if c["score"] == "softmax":
        scores = scores / scores.sum(1, keepdim=True)
    wanted = scores if s["bias"] is None else scores + s["bias"].double()
    ids = torch.sort(wanted, dim=1, descending=True, stable=True).indices[:, :c["top"]]
    weights = scores.gather(1, ids)
    if c["normalise"]:
        weights = weights / weights.sum(1, keepdim=True)
    return ids.int(), (weights * c["factor"]).float()


def _experts_plain(s):
    c, d = s["case"], s["x"].dtype
    ids, weights = _route_plain(s)
    t, k, f, e, top = c["tokens"], c["k"], c["hidden"], c["experts"], c["top"]
    x, chosen = s["x"].float(), ids.long()
    if t * top < e:  # the chosen experts' weights, once a choice
        at = chosen.flatten()
        rows = x.repeat_interleave(top, 0)[:, :, None]
        both = torch.bmm(s["gate_up"][at].float(), rows)[..., 0] * s["gate_up_scale"][at]
        gate, up = both[:, :f], both[:, f:]
        hidden = gate / (1 + torch.exp(-gate)) * up
        out = (torch.bmm(s["down"][at].float(), hidden[:, :, None])[..., 0] * s["down_scale"][at]).view(t, top, k)
    else:  # every expert over every token
        both = torch.bmm(s["gate_up"].float(), x.T.contiguous().expand(e, k, t).contiguous()) * s["gate_up_scale"][..., None]
        gate, up = both[:, :f], both[:, f:]
        hidden = gate / (1 + torch.exp(-gate)) * up
        out = torch.bmm(s["down"].float(), hidden) * s["down_scale"][..., None]
        out = out.permute(2, 0, 1)[torch.arange(t, device=DEVICE)[:, None], chosen]
    total = (out * weights[..., None]).sum(1)
    if s["residual"] is not None:
        total = total + s["residual"].float()
    return {"ids": ids, "weights": weights, "out": total.to(d)}


def _sample_plain(s):
    options = {name: torch.as_tensor(value, device=DEVICE).double().expand(len(s["logits"]))[:, None] for name, value in s["options"].items()}
    logits = s["logits"].double()
    ordered, index = torch.sort(logits, dim=1, descending=True, stable=True)
    warm = options["temperature"] > 0
    weight = torch.exp((ordered - ordered[:, :1]) / torch.where(warm, options["temperature"], 1.0))
    place = torch.arange(logits.shape[1], device=DEVICE)[None]
    kept = (options["top_k"] <= 0) | (place < options["top_k"])
    mass = torch.cumsum(weight * kept, 1)
    before = mass - weight * kept
    kept = kept & ((options["top_p"] >= 1) | (before < options["top_p"] * mass[:, -1:]) | (place == 0))
    kept = kept & (weight >= options["min_p"])
    left = torch.zeros_like(weight).scatter_(1, index, weight * kept)
    upto = torch.cumsum(left, 1)
    drawn = (upto > s["draws"].double()[:, None] * upto[:, -1:]).int().argmax(1)
    return {"tokens": torch.where(warm[:, 0], drawn, index[:, 0])}


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    s, c = state, state["case"]
    if not own:
        return {"add": _add_plain, "experts": _experts_plain, "sample": _sample_plain}[c["op"]](s)
    from wgpkernels_amd import int8 as wq
    if c["op"] == "add":
        prepared, total = wq.add_prepare(s["x"], s["residual"], s["scale"], group=c["rotation"], path=c["path"], act_weight=s["weight"], eps=EPS)
        return {"sum": total, "values": prepared.values()}
    if c["op"] == "experts":
        routes = wq.route(s["x"], s["router"], c["top"], score=c["score"], bias=s["bias"], normalise=c["normalise"], factor=c["factor"])
        out = wq.experts(s["x"], routes, s["gate_up"], s["gate_up_scale"], s["down"], s["down_scale"], residual=s["residual"])
        return {"ids": routes.ids, "weights": routes.weights, "out": out}
    return {"tokens": wq.sample(s["logits"], s["draws"], **s["options"])}


# ---- 64 bits, from the definitions ----------------------------------------------------------------------------------
def _exact_add(c, s):
    scale = torch.ones(c["k"], device=DEVICE) if s["scale"] is None else s["scale"]
    total = torch.addcmul(s["residual"].double(), s["x"].double(), scale.double())
    held = total.float().to(s["x"].dtype).double()
    v = held * torch.rsqrt(torch.linalg.vector_norm(held, dim=1, keepdim=True) ** 2 / c["k"] + EPS)
    v = v * (1.0 if s["weight"] is None else s["weight"].double())
    if c["rotation"]:  # digit by digit, from the fastest one
        places = v.view(len(v), -1, *[4] * round(math.log(c["rotation"], 4)))
        for axis in range(2, places.dim()):
            places = (places.sum(axis, keepdim=True) - 2 * places.flip(axis)) / 2
        v = places.reshape(v.shape)
    if c["path"] == "small":
        return {"sum": total, "values": v}
    parts = v.split(128, 1) if c["path"] == "block" else [v]
    found = []
    for part in parts:
        top = part.abs().amax(1, keepdim=True)
        unit = torch.where(top > 0, 127 / top, 0.0)
        code = torch.round(part * unit)
        rest = torch.round((part * unit - code) * 254) / 254 if c["path"] == "exact" else 0.0
        found.append((code + rest) * top / 127)
    return {"sum": total, "values": torch.cat(found, 1)}


def _exact_experts(c, s):
    x = s["x"].double()
    logits = torch.stack([(x * row.double()).sum(1) for row in s["router"]], 1)
    scores = torch.softmax(logits, 1) if c["score"] == "softmax" else torch.sigmoid(logits)
    ids = torch.argsort(scores + (0.0 if s["bias"] is None else s["bias"].double()), dim=1, descending=True, stable=True)[:, :c["top"]]
    weights = torch.gather(scores, 1, ids) * c["factor"]
    if c["normalise"]:
        weights = weights / torch.gather(scores, 1, ids).sum(1, keepdim=True)
    total = torch.zeros_like(x) if s["residual"] is None else s["residual"].double()
    for e in range(c["experts"]):
        token, place = torch.nonzero(ids == e, as_tuple=True)
        if len(token):
            rows = x[token] @ (s["gate_up"][e].double() * s["gate_up_scale"][e].double()[:, None]).T
            gate, up = rows.split(c["hidden"], 1)
            out = (gate * torch.sigmoid(gate) * up) @ (s["down"][e].double() * s["down_scale"][e].double()[:, None]).T
            total.index_add_(0, token, out * weights[token, place][:, None])
    return {"ids": ids.int(), "weights": weights, "out": total}


def exact(case, seed):
    c = {k: v for k, v in case.items() if k != "name"}
    if c["op"] == "sample":
        return None
    return {"add": _exact_add, "experts": _exact_experts}[c["op"]](c, _inputs(c, seed))
