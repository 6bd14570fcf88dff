"""What is measured of the operators around the decode layer, and on which inputs.

Four operators, as one step of a decoder with expert layers uses them in turn:

* ``norm``      residual addition and root-mean-square norm, result in BF16
* ``norm_fp8``  the same with the result as E4M3 codes and one FP32 scale per row
* ``layer``     router, top-k, experts and weighted sum for at most eight tokens, expert
                weights in BF16 or in E4M3 with one scale per row
* ``sample``    one token per row of logits: temperature, top-k, top-p and min-p, with the
                random numbers given

``run`` computes them in elementary torch operations, or, where ``own`` is set, by the
package's entry points.
"""

import math
import os
import sys

import numpy as np
import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "b300-moe-decode-fastpath_b200")
_api = None


def _package():
    """The package, imported when the first call of it is made (and then kept)."""
    global _api
    if _api is None:
        for folder in (os.path.join(os.getcwd(), "b300-moe-decode-fastpath_b200"), _PACKAGE):
            if os.path.isdir(folder) and folder not in sys.path:
                sys.path.insert(0, folder)
        import b200moe
        _api = b200moe
    return _api


# ---------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------
def listed():
    return [
        # one token of one request: the norm in front of the expert layer, all latency
        {"name": "norm 1x4096", "op": "norm", "rows": 1, "hidden": 4096,
         "residual": "bf16", "weight": "bf16"},
        # a prompt of 8192 tokens with the residual stream kept in BF16: all bandwidth
        {"name": "norm 8192x4096", "op": "norm", "rows": 8192, "hidden": 4096,
         "residual": "bf16", "weight": "bf16"},
        # a full decode batch with an FP32 residual stream, result in 8 bits
        {"name": "norm fp8 64x7168", "op": "norm_fp8", "rows": 64, "hidden": 7168,
         "residual": "fp32", "weight": "fp32"},
        # a packed batch of prompts whose lengths add up to an odd number
        {"name": "norm fp8 4099x2880", "op": "norm_fp8", "rows": 4099, "hidden": 2880,
         "residual": "bf16", "weight": "bf16"},
        # one token through many small experts: the call where fixed costs count most
        {"name": "layer 1 token, 128 experts of 768", "op": "layer", "tokens": 1,
         "hidden": 2048, "inter": 768, "experts": 128, "top_k": 8, "kind": "bf16",
         "router": "bf16", "routing": False},
        # a small batch through the same layer: most experts have one token
        {"name": "layer 8 tokens, 128 experts of 768", "op": "layer", "tokens": 8,
         "hidden": 2048, "inter": 768, "experts": 128, "top_k": 8, "kind": "bf16",
         "router": "fp32", "routing": True},
        # the Mixtral-shaped layer with every expert in use: the most bytes
        {"name": "layer 8 tokens, 8 experts of 14336", "op": "layer", "tokens": 8,
         "hidden": 4096, "inter": 14336, "experts": 8, "top_k": 2, "kind": "bf16",
         "router": "bf16", "routing": False},
        # the irregular layer (no size a power of two) with E4M3 weights
        {"name": "layer fp8 3 tokens, 32 experts of 2880", "op": "layer", "tokens": 3,
         "hidden": 2880, "inter": 2880, "experts": 32, "top_k": 8, "kind": "fp8",
         "router": "bf16", "routing": True},
        # one request, nucleus sampling
        {"name": "sample 1x32000", "op": "sample", "rows": 1, "vocab": 32000, "pad": 0,
         "dtype": "fp32", "spread": 2.5, "filters": "p", "logprobs": False},
        # requests with settings of their own over a large vocabulary
        {"name": "sample 64x129280", "op": "sample", "rows": 64, "vocab": 129280, "pad": 0,
         "dtype": "fp32", "spread": 2.5, "filters": "mixed", "logprobs": True},
        # an odd vocabulary in padded rows of BF16 logits, top-k then top-p
        {"name": "sample 17x32003 bf16", "op": "sample", "rows": 17, "vocab": 32003, "pad": 61,
         "dtype": "bf16", "spread": 2.5, "filters": "kp", "logprobs": False},
        # plain temperature sampling from nearly flat rows: every token has to be weighed
        {"name": "sample 8x129280 flat", "op": "sample", "rows": 8, "vocab": 129280, "pad": 0,
         "dtype": "fp32", "spread": 0.5, "filters": "none", "logprobs": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(("norm", "norm_fp8", "layer", "layer", "sample", "sample"))
    if op in ("norm", "norm_fp8"):
        step = 8 if op == "norm" else 16
        hidden = max(1, _log(rng, 64, 16384) // step) * step
        rows = min(_log(rng, 1, 8192), 8192 * 4096 // hidden)
        return {"op": op, "rows": rows, "hidden": hidden,
                "residual": rng.choice(("bf16", "bf16", "fp32", "none")),
                "weight": rng.choice(("bf16", "fp32"))}
    if op == "layer":
        kind = rng.choice(("bf16", "fp8"))
        step = 8 if kind == "bf16" else 16
        top_k = rng.choice((1, 2, 4, 8))
        experts = _log(rng, max(top_k, 2), 256)
        tokens = rng.randint(1, 8)
        hidden = max(1, _log(rng, 256, 7168) // step) * step
        # at most the expert weights, and the weight rows in use, of the largest listed case
        most = min(8 * 4096 * 14336 // (experts * hidden),
                   16 * 4096 * 14336 // (tokens * top_k * hidden), 14336)
        inter = max(step, _log(rng, 64, max(64, most)) // step * step)
        return {"op": "layer", "tokens": tokens, "hidden": hidden, "inter": inter,
                "experts": experts, "top_k": top_k, "kind": kind,
                "router": rng.choice(("bf16", "fp32")), "routing": rng.random() < 0.5}
    rows = _log(rng, 1, 64)
    vocab = _log(rng, 200, 129280)
    return {"op": "sample", "rows": rows, "vocab": vocab, "pad": rng.choice((0, 0, 1, 61)),
            "dtype": rng.choice(("bf16", "fp32")), "spread": rng.choice((0.5, 2.5, 6.0)),
            "filters": rng.choice(("none", "p", "k", "kp", "mixed")),
            "logprobs": rng.random() < 0.5}


_TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp32": 4, "none": 0}


def work(case):
    op = case["op"]
    if op in ("norm", "norm_fp8"):
        n = case["rows"] * case["hidden"]
        size = 2 * n + 2 * _SIZE[case["residual"]] * n + case["hidden"] * _SIZE[case["weight"]]
        size += 2 * n if op == "norm" else n + 4 * case["rows"]
        return {"bytes": size, "flops": 5 * n}
    if op == "layer":
        t, h, i = case["tokens"], case["hidden"], case["inter"]
        e, k = case["experts"], case["top_k"]
        used = e * (1.0 - (1.0 - k / e) ** t)  # experts in use, on average
        each = 3 * h * i * (2 if case["kind"] == "bf16" else 1)
        if case["kind"] == "fp8":
            each += 4 * (2 * i + h)
        size = used * each + e * h * _SIZE[case["router"]] + 4 * t * h
        return {"bytes": size, "flops": 6 * t * k * h * i + 2 * t * e * h}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * _SIZE[case["dtype"]] + 32 * case["rows"], "flops": 4 * n}


# ---------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _prepare_norm(case, g):
    rows, hidden = case["rows"], case["hidden"]
    x = _normal(g, rows, hidden)
    residual = None
    if case["residual"] != "none":
        residual = _normal(g, rows, hidden, std=3.0, dtype=_TYPES[case["residual"]])
    weight = (1.0 + _normal(g, hidden, std=0.1, dtype=torch.float32)).to(_TYPES[case["weight"]])
    # the buffers a decode loop keeps from step to step
    out = torch.empty(rows, hidden, device="cuda",
                      dtype=torch.bfloat16 if case["op"] == "norm" else torch.uint8)
    return {"x": x, "residual": residual, "weight": weight, "eps": 1e-6, "out": out,
            "scale": torch.empty(rows, device="cuda"),
            "residual_out": None if residual is None else torch.empty_like(residual)}


def _codes(g, *shape):
    return _normal(g, *shape, std=100.0).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)


def _scales(g, *shape, std):
    return torch.empty(*shape, device="cuda").uniform_(0.8, 1.25, generator=g) * (std / 100.0)


def _prepare_layer(case, g):
    t, h, i, e = case["tokens"], case["hidden"], case["inter"], case["experts"]
    state = {
        "x": _normal(g, t, h),
        "router": _normal(g, e, h, std=h ** -0.5, dtype=_TYPES[case["router"]]),
        "experts": e, "top_k": case["top_k"], "routing": case["routing"], "kind": case["kind"],
        "out": torch.empty(t, h, dtype=torch.bfloat16, device="cuda"),
    }
    if case["kind"] == "bf16":
        state["gate_up"] = _normal(g, e, 2 * i, h, std=h ** -0.5)
        state["down"] = _normal(g, e, h, i, std=i ** -0.5)
    else:
        state["gate_up"] = _codes(g, e, 2 * i, h)
        state["gate_up_scale"] = _scales(g, e, 2 * i, std=h ** -0.5)
        state["down"] = _codes(g, e, h, i)
        state["down_scale"] = _scales(g, e, h, std=i ** -0.5)
    if own:  # the handle that a program keeps: scratch memory and the weights' record
        api = _package()
        state["workspace"] = api.B300MoEWorkspace(t, device="cuda")
        if case["kind"] == "fp8":
            state["weights"] = api.Fp8ExpertWeights(state["gate_up"], state["gate_up_scale"],
                                                    state["down"], state["down_scale"])
    return state


def _prepare_sample(case, g):
    rows, vocab = case["rows"], case["vocab"]
    held = _normal(g, rows, vocab + case["pad"], std=case["spread"], dtype=torch.float32)
    # a few tokens that the model favours, and a grammar that forbids some
    favoured = torch.randint(0, vocab, (rows, 8), generator=g, device="cuda")
    held.scatter_add_(1, favoured, torch.full((rows, 8), 2.0 * case["spread"], device="cuda"))
    forbidden = torch.randint(0, vocab, (rows, vocab // 16), generator=g, device="cuda")
    held.scatter_(1, forbidden, float("-inf"))
    u = torch.rand(rows, generator=g, device="cuda")
    row = torch.arange(rows, device="cuda")
    temperature = 0.6 + 0.1 * (row % 7).float()
    top_k = torch.zeros(rows, dtype=torch.int32, device="cuda")
    top_p = torch.ones(rows, device="cuda")
    min_p = torch.zeros(rows, device="cuda")
    if case["filters"] in ("p", "kp"):
        top_p = 0.8 + 0.05 * (row % 4).float()
    if case["filters"] in ("k", "kp"):
        top_k = (20 + 30 * (row % 3)).to(torch.int32)
    if case["filters"] == "mixed":
        # requests in turn: greedy, plain, nucleus, top-k, both, min-p, all three
        mode = row % 7
        temperature = torch.where(mode == 0, torch.zeros_like(temperature), temperature)
        top_p = torch.where((mode == 2) | (mode == 4) | (mode == 6), 0.9, top_p)
        top_k = torch.where((mode == 3) | (mode == 4) | (mode == 6), 50, top_k).to(torch.int32)
        min_p = torch.where(mode >= 5, 0.05, min_p)
    return {"logits": held.to(_TYPES[case["dtype"]])[:, :vocab], "u": u,
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "logprobs": case["logprobs"]}


def prepare(case, seed):
    g = _generator(seed)
    make = {"norm": _prepare_norm, "norm_fp8": _prepare_norm, "layer": _prepare_layer,
            "sample": _prepare_sample}[case["op"]]
    state = make(case, g)
    state["op"] = case["op"]
    return state


# ---------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------
def _plain_norm(s):
    total = s["x"].float()
    if s["residual"] is not None:
        total = total + s["residual"].float()
    y = total * torch.rsqrt(total.square().mean(-1, keepdim=True) + s["eps"]) * s["weight"].float()
    kept = {} if s["residual"] is None else {"residual": total.to(s["residual"].dtype)}
    if s["op"] == "norm":
        return {"out": y.to(torch.bfloat16), **kept}
    largest = y.abs().amax(-1)
    scale = torch.where(largest > 0, largest / 448.0, torch.ones_like(largest))
    return {"out": (y / scale[:, None]).to(torch.float8_e4m3fn), "scale": scale, **kept}


def _plain_layer(s):
    x, k = s["x"], s["top_k"]
    # the logits in 64 bits: two experts may lie next to one another at the border
    logits = x.double() @ s["router"].double().T
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    ids = order.indices[:, :k]
    weights = torch.softmax(order.values[:, :k], dim=-1).float()

    def rows(name):  # [T, K, rows, columns] in FP32
        held = s[name][ids]
        if s["kind"] == "bf16":
            return held.float()
        return held.view(torch.float8_e4m3fn).float() * s[name + "_scale"][ids][..., None]

    both = (rows("gate_up") @ x.float()[:, None, :, None]).squeeze(-1)
    gate, up = both.chunk(2, dim=-1)
    act = gate / (1.0 + torch.exp(-gate)) * up
    each = (rows("down") @ act[..., None]).squeeze(-1)
    out = (each * weights[..., None]).sum(1).to(torch.bfloat16)
    return {"out": out, "ids": ids, "weights": weights} if s["routing"] else {"out": out}


def _plain_sample(s):
    x = s["logits"].float()
    x = torch.where(x.isnan(), float("-inf"), x)
    vocab = x.shape[1]
    # sums and products in 64 bits: with a large vocabulary the borders between tokens lie
    # closer together than 32 bits resolve
    values, order = torch.sort(x, dim=-1, descending=True, stable=True)
    best = values[:, :1]
    temperature = s["temperature"][:, None].double()
    below = torch.where(values == best, 0.0, values.double() - best.double())
    w = torch.exp(below / torch.where(temperature > 0, temperature, 1.0))
    rank = torch.arange(vocab, device=x.device)[None]
    top_k, top_p, min_p = s["top_k"][:, None], s["top_p"][:, None].double(), s["min_p"][:, None].double()
    keep = (values > float("-inf")) & ((top_k <= 0) | (rank < top_k)) & (w >= min_p.clamp(max=1.0))
    w = torch.where(keep, w, 0.0)
    before = torch.cumsum(w, -1) - w
    total = w.sum(-1, keepdim=True)
    keep = keep & ((top_p >= 1) | (before < top_p * total) | (rank == 0))
    w = torch.zeros_like(w).scatter(1, order, torch.where(keep, w, 0.0))  # in the tokens' order
    upto = torch.cumsum(w, -1)
    total = upto[:, -1:]
    last = (vocab - 1 - (w.flip(-1) > 0).int().argmax(-1, keepdim=True)).clamp(min=0)
    pick = (upto <= s["u"][:, None].double() * total).sum(-1, keepdim=True).minimum(last)
    logp = torch.log(w.gather(1, pick) / total)
    greedy = ~(temperature > 0)
    pick, logp = torch.where(greedy, order[:, :1], pick), torch.where(greedy, 0.0, logp)
    none = best == float("-inf")
    pick, logp = torch.where(none, -1, pick), torch.where(none, float("-inf"), logp)
    return {"ids": pick[:, 0], "logprobs": logp[:, 0].float()} if s["logprobs"] else {"ids": pick[:, 0]}


def _own_norm(s):
    api = _package()
    if s["op"] == "norm":
        out, residual = api.add_rms_norm(s["x"], s["residual"], s["weight"], eps=s["eps"],
                                         out=s["out"], residual_out=s["residual_out"])
        got = {"out": out}
    else:
        codes, scale, residual = api.add_rms_norm_fp8(
            s["x"], s["residual"], s["weight"], eps=s["eps"], out=s["out"],
            scale_out=s["scale"], residual_out=s["residual_out"])
        got = {"out": codes.view(torch.float8_e4m3fn), "scale": scale}
    if s["residual"] is not None:
        got["residual"] = residual
    return got


def _own_layer(s):
    api = _package()
    options = {"num_experts": s["experts"], "top_k": s["top_k"], "workspace": s["workspace"],
               "return_routing": s["routing"], "out": s["out"]}
    if s["kind"] == "bf16":
        got = api.b300_moe_layer(s["x"], s["router"], s["gate_up"], s["down"], **options)
    else:
        got = api.b300_moe_layer_fp8(s["x"], s["router"], s["weights"], **options)
    return dict(zip(("out", "ids", "weights"), got)) if s["routing"] else {"out": got}


def _own_sample(s):
    got = _package().sample_tokens(
        s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
        min_p=s["min_p"], return_logprobs=s["logprobs"])
    return dict(zip(("ids", "logprobs"), got)) if s["logprobs"] else {"ids": got}


def run(state):
    op = state["op"]
    if own:
        return (_own_layer if op == "layer" else _own_sample if op == "sample" else _own_norm)(state)
    return (_plain_layer if op == "layer" else _plain_sample if op == "sample" else _plain_norm)(state)


# ---------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------
def _exact_norm(case, s):
    sums = s["x"].double() + (0.0 if s["residual"] is None else s["residual"].double())
    length = torch.sqrt((sums * sums).sum(-1, keepdim=True) / case["hidden"] + s["eps"])
    y = sums / length * s["weight"].double()
    kept = {} if s["residual"] is None else {"residual": sums}
    if case["op"] == "norm":
        return {"out": y, **kept}
    scale = y.abs().max(-1).values / 448.0
    scale[scale == 0] = 1.0
    return {"out": y / scale[:, None], "scale": scale, **kept}


def _exact_layer(case, s):
    t, h, k = case["tokens"], case["hidden"], case["top_k"]
    x = s["x"].double()
    logits = torch.stack([(s["router"].double() * row).sum(-1) for row in x]).cpu().numpy()
    ids = np.argsort(-logits, axis=1, kind="stable")[:, :k]
    chosen = np.take_along_axis(logits, ids, 1)
    weights = np.exp(chosen - chosen.max(1, keepdims=True))
    weights /= weights.sum(1, keepdims=True)
    out = torch.zeros(t, h, dtype=torch.float64, device="cuda")
    for e in np.unique(ids):
        def matrix(name):
            if case["kind"] == "bf16":
                return s[name][e].double()
            return s[name][e].view(torch.float8_e4m3fn).double() * s[name + "_scale"][e].double()[:, None]
        gate_up, down = matrix("gate_up"), matrix("down")
        for row, slot in zip(*np.nonzero(ids == e)):
            both = gate_up @ x[row]
            gate, up = both[:case["inter"]], both[case["inter"]:]
            out[row] += float(weights[row, slot]) * (down @ (gate * torch.sigmoid(gate) * up))
    if not case["routing"]:
        return {"out": out}
    return {"out": out, "ids": torch.from_numpy(ids.copy()), "weights": torch.from_numpy(weights)}


def _exact_sample(case, s):
    logits = s["logits"].double().cpu().numpy()
    settings = [s[name].double().cpu().numpy() for name in ("u", "temperature", "top_k", "top_p", "min_p")]
    ids, logprobs = [], []
    for x, u, temperature, top_k, top_p, min_p in zip(logits, *settings):
        x = np.where(np.isnan(x), -np.inf, x)
        best = x.max()
        if best == -np.inf:
            ids.append(-1)
            logprobs.append(-np.inf)
            continue
        if not temperature > 0:
            ids.append(int(x.argmax()))
            logprobs.append(0.0)
            continue
        order = np.argsort(-x, kind="stable")
        order = order[x[order] > -np.inf]
        if top_k > 0:
            order = order[:int(top_k)]
        w = np.exp(np.where(x[order] == best, 0.0, x[order] - best) / temperature)
        order, w = order[w >= min(min_p, 1.0)], w[w >= min(min_p, 1.0)]
        if top_p < 1:
            count = int(np.searchsorted(np.cumsum(w), top_p * w.sum())) + 1
            order, w = order[:count], w[:count]
        place = np.argsort(order)
        order, w = order[place], w[place]
        upto = np.cumsum(w)
        at = min(int(np.searchsorted(upto, u * upto[-1], side="right")), len(w) - 1)
        ids.append(int(order[at]))
        logprobs.append(float(np.log(w[at] / upto[-1])))
    got = {"ids": torch.tensor(ids, dtype=torch.int64)}
    if case["logprobs"]:
        got["logprobs"] = torch.tensor(logprobs, dtype=torch.float64)
    return got


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "layer":
        return _exact_layer(case, state)
    if case["op"] == "sample":
        return _exact_sample(case, state)
    return _exact_norm(case, state)
