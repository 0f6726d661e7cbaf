"""What the mixture-of-experts operators are measured on: cases, inputs, the operators' plain form and their exact values.

Four operators over 4-bit affine experts (codes 0..15, one bf16 scale and bias per 64 inputs, w = scale * q + bias):

  route    logits [M, E] -> the k experts of every row, their weights, and the (row, place) pairs sorted by expert
  grouped  y[m, j] = W[ids[m, j]] x[m]: one product per expert over the ragged set of rows that chose it
  experts  y[m, j] = D[e] (act(G[e] x[m]) * (U[e] x[m])), e = ids[m, j]: an expert's gated MLP
  block    h' = scale * h + gate * norm(sum_j w[m, j] y[m, j]);  z = norm(h'): the block's output joins the residual
           stream, and the next block's input is normalised

`run` computes them with elementary torch operations in 32 bits, or, where `own` is true, through ironmule_b200.
"""
from __future__ import annotations

import math

import torch

own = False

GROUP = 64
EPS = 1e-6


# ---- cases ----------------------------------------------------------------------------------------------------
def _route(name, rows, experts, top_k, dtype="bf16", scoring="softmax", normalise=True, scale=1.0, bias=False,
           closed=0.0):
    return {"name": name, "op": "route", "rows": rows, "experts": experts, "top_k": top_k, "dtype": dtype,
            "scoring": scoring, "normalise": normalise, "scale": scale, "bias": bias, "closed": closed}


def _experts(name, rows, experts, top_k, hidden, inter, act="swiglu", skew=0.3):
    return {"name": name, "op": "experts", "rows": rows, "experts": experts, "top_k": top_k, "hidden": hidden,
            "inter": inter, "act": act, "skew": skew}


def _grouped(name, rows, experts, top_k, n, k, closed=0.0, skew=0.3):
    return {"name": name, "op": "grouped", "rows": rows, "experts": experts, "top_k": top_k, "n": n, "k": k,
            "closed": closed, "skew": skew}


def _block(name, rows, places, hidden, post=False, gate="none", res_scale=1.0, gemma=False, closed=0.0):
    return {"name": name, "op": "block", "rows": rows, "places": places, "hidden": hidden, "post": post, "gate": gate,
            "res_scale": res_scale, "gemma": gemma, "closed": closed}


def listed():
    return [
        # one decoded token: latency is everything
        _route("route-token", 1, 128, 8),
        # a long prompt's prefill in one piece
        _route("route-prefill", 8192, 128, 8),
        # an odd batch over an odd number of experts, scored by sigmoid with a balancing bias, a tenth of the
        # experts closed to each row (capacity or expert-parallel masks), rows without any expert among them
        _route("route-masked", 333, 60, 4, dtype="f32", scoring="sigmoid", scale=2.5, bias=True, closed=0.1),
        # one decoded token through its eight experts: matrix-vector products over 4-bit weights
        _experts("experts-token", 1, 128, 8, 2048, 768),
        # one speculative verification pass: four drafted tokens and the target's own
        _experts("experts-verify", 5, 128, 8, 2048, 768),
        # a verification pass of 32 sequences: every expert is chosen, by ten rows on average
        _experts("experts-batch", 160, 128, 8, 2048, 768),
        # a prompt's prefill: about 256 rows an expert, unevenly
        _experts("experts-prefill", 4096, 128, 8, 2048, 768),
        # few wide experts (the dense 2560 x 9728 MLP of the benchmarked target, eight times), an odd batch
        _experts("experts-wide", 91, 8, 2, 2560, 9728, act="geglu"),
        # a projection by expert at awkward sizes: outputs that fill no tile, experts without rows, closed places
        _grouped("grouped-odd", 77, 60, 4, 1000, 576, closed=0.2, skew=1.5),
        # a projection by expert over a prompt
        _grouped("grouped-prompt", 1500, 32, 4, 2560, 1024),
        # one decoded token's experts joined, the residual added, the next norm taken
        _block("block-token", 1, 8, 2048),
        # a prefill's, with the output norm and a learned gate a channel
        _block("block-prefill", 4096, 8, 2048, post=True, gate="channel", res_scale=0.5),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["route", "experts", "experts", "grouped", "block"])
    if op == "route":
        experts = _log_int(rng, 4, 256)
        return _strip(_route("", _log_int(rng, 1, 8192), experts, rng.randint(1, min(8, experts)),
                             dtype=rng.choice(["bf16", "f32"]), scoring=rng.choice(["softmax", "sigmoid"]),
                             normalise=rng.random() < 0.7, scale=rng.choice([1.0, 2.5]), bias=rng.random() < 0.5,
                             closed=rng.choice([0.0, 0.1, 0.6])))
    if op == "block":
        hidden = 64 * _log_int(rng, 4, 84)
        places = rng.randint(1, 8)
        rows = _log_int(rng, 1, 4096)
        rows = max(1, min(rows, 4096 * 8 * 2048 // (places * hidden)))
        return _strip(_block("", rows, places, hidden, post=rng.random() < 0.5,
                             gate=rng.choice(["none", "channel", "row", "full"]), res_scale=rng.choice([1.0, 0.5]),
                             gemma=rng.random() < 0.5, closed=rng.choice([0.0, 0.2])))
    experts = _log_int(rng, 4, 128)
    top_k = rng.randint(1, min(8, experts))
    if op == "experts":
        hidden, inter = 64 * _log_int(rng, 4, 40), 64 * _log_int(rng, 2, 40)
        while experts > 4 and experts * 3 * hidden * inter > 128 * 3 * 2048 * 768:
            experts //= 2
        top_k = min(top_k, experts)
        rows = _log_int(rng, 1, 4096)
        rows = max(1, min(rows, 4096 * 8 * 2048 * 768 // (top_k * hidden * inter)))
        return _strip(_experts("", rows, experts, top_k, hidden, inter, act=rng.choice(["swiglu", "geglu"]),
                               skew=rng.choice([0.0, 0.3, 1.5])))
    n, k = _log_int(rng, 100, 4096), 64 * _log_int(rng, 2, 40)
    while experts > 4 and experts * n * k > 128 * 3 * 2048 * 768:
        experts //= 2
    top_k = min(top_k, experts)
    rows = _log_int(rng, 1, 4096)
    rows = max(1, min(rows, 4096 * 8 * 2048 * 1024 // (top_k * n * k)))
    return _strip(_grouped("", rows, experts, top_k, n, k, closed=rng.choice([0.0, 0.2]),
                           skew=rng.choice([0.0, 0.3, 1.5])))


def _strip(case):
    del case["name"]
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(gen, *shape, std=1.0):
    return torch.randn(shape, generator=gen, device="cuda") * std


def _quantised(gen, experts, n, k):
    """Random 4-bit affine matrices [E, N, K] with entries of about 0.02 around zero."""
    w = torch.randint(-2**31, 2**31, (experts, n, k // 8), generator=gen, device="cuda", dtype=torch.int64)
    scales = 0.0043 * (0.5 + torch.rand((experts, n, k // GROUP), generator=gen, device="cuda"))
    biases = -7.5 * scales + _normal(gen, experts, n, k // GROUP, std=0.002)
    return w.to(torch.int32), scales.to(torch.bfloat16), biases.to(torch.bfloat16)


def _logits(gen, case):
    """Router outputs: unit spread over the experts of a row, some experts more popular than others. A share
    `closed` of the places is masked with -inf; one row in eight of a masked batch loses every expert."""
    rows, experts = case["rows"], case["experts"]
    logits = _normal(gen, rows, experts) + _normal(gen, experts, std=case.get("skew", 0.3))
    closed = case.get("closed", 0.0)
    if closed:
        mask = torch.rand((rows, experts), generator=gen, device="cuda") < closed
        mask |= torch.rand((rows, 1), generator=gen, device="cuda") < 0.125
        logits = logits.masked_fill(mask, float("-inf"))
    return logits.to(torch.float32 if case.get("dtype") == "f32" else torch.bfloat16)


def _inputs(case, seed):
    gen = _gen(seed)
    op = case["op"]
    if op == "block":
        rows, places, hidden = case["rows"], case["places"], case["hidden"]
        weights = torch.softmax(_normal(gen, rows, places), dim=1)
        closed = torch.rand((rows, places), generator=gen, device="cuda") < case["closed"]
        base = 0.0 if case["gemma"] else 1.0
        shape = {"none": None, "channel": (hidden,), "row": (rows, 1), "full": (rows, hidden)}[case["gate"]]
        return {"y": _normal(gen, rows, places, hidden, std=0.5).to(torch.bfloat16),
                "weights": weights.masked_fill(closed, 0.0),
                "h": _normal(gen, rows, hidden, std=2.0).to(torch.bfloat16),
                "post": (base + _normal(gen, hidden, std=0.1)).to(torch.bfloat16) if case["post"] else None,
                "gate": (0.5 + _normal(gen, *shape, std=0.2)).to(torch.bfloat16) if shape else None,
                "next": (base + _normal(gen, hidden, std=0.1)).to(torch.bfloat16)}
    state = {"logits": _logits(gen, case)}
    if op == "route":
        state["bias"] = _normal(gen, case["experts"], std=0.2) if case["bias"] else None
    elif op == "grouped":
        state["x"] = _normal(gen, case["rows"], case["k"]).to(torch.bfloat16)
        state["w"] = _quantised(gen, case["experts"], case["n"], case["k"])
    else:
        hidden, inter = case["hidden"], case["inter"]
        state["x"] = _normal(gen, case["rows"], hidden).to(torch.bfloat16)
        state["gate"] = _quantised(gen, case["experts"], inter, hidden)
        state["up"] = _quantised(gen, case["experts"], inter, hidden)
        state["down"] = _quantised(gen, case["experts"], hidden, inter)
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if own and case["op"] in ("grouped", "experts"):
        from ironmule_b200 import kernels

        # the resident weights of such a program: repacked once
        if case["op"] == "grouped":
            state["packed"] = kernels.Experts(*state.pop("w"))
        else:
            state["packed"] = (kernels.Experts.gate_up(state.pop("gate"), state.pop("up")),
                               kernels.Experts(*state.pop("down")))
    return state


# ---- the plain form -------------------------------------------------------------------------------------------
def _plain_route(logits, top_k, scoring="softmax", normalise=True, scale=1.0, bias=None):
    rows, experts = logits.shape
    values = logits.float()
    values = torch.where(torch.isnan(values), float("-inf"), values)
    keys = values if bias is None else values + bias
    order = torch.sort(keys, dim=1, descending=True, stable=True).indices[:, :top_k]
    chosen = torch.gather(values, 1, order)
    opened = chosen > float("-inf")
    if scoring == "softmax":
        top = values.amax(dim=1, keepdim=True)
        top = torch.where(top > float("-inf"), top, 0.0)
        weights = torch.exp(chosen - top)
        total = weights.sum(dim=1, keepdim=True) if normalise else torch.exp(values - top).sum(dim=1, keepdim=True)
        weights = weights / total
    else:
        weights = 1.0 / (1.0 + torch.exp(-chosen))
        if normalise:
            weights = weights / weights.sum(dim=1, keepdim=True)
    weights = torch.where(opened, weights * scale, 0.0)
    ids = torch.where(opened, order, -1).to(torch.int32)
    buckets = torch.where(ids < 0, experts, ids).flatten()
    pairs = torch.sort(buckets, stable=True).indices.to(torch.int32)
    counts = (buckets[:, None] == torch.arange(experts + 1, device=logits.device)).sum(dim=0)
    offsets = torch.nn.functional.pad(torch.cumsum(counts, 0), (1, 0)).to(torch.int32)
    return ids, weights, offsets, pairs


def _plain_dense(w, scales, biases):
    """One expert's matrix [N, K] in 32 bits."""
    shifts = torch.arange(0, 32, 4, device=w.device, dtype=torch.int32)
    q = ((w[:, :, None] >> shifts) & 15).reshape(w.shape[0], -1, GROUP).float()
    return (scales.float()[:, :, None] * q + biases.float()[:, :, None]).reshape(w.shape[0], -1)


def _plain_act(gate, act):
    if act == "swiglu":
        return gate / (1.0 + torch.exp(-gate))
    return 0.5 * gate * (1.0 + torch.tanh(0.7978845608028654 * (gate + 0.044715 * gate * gate * gate)))


def _plain_by_expert(ids, experts, width, compute):
    rows, top_k = ids.shape
    flat = ids.flatten()
    y = torch.zeros((rows * top_k, width), dtype=torch.bfloat16, device=ids.device)
    for e in range(experts):
        pair = (flat == e).nonzero()[:, 0]
        if pair.numel():
            y[pair] = compute(e, pair // top_k).to(torch.bfloat16)
    return y.view(rows, top_k, width)


def _plain_norm(v, weight, gemma):
    factor = 1.0 + weight.float() if gemma else weight.float()
    return v / torch.sqrt((v * v).mean(dim=1, keepdim=True) + EPS) * factor


def _plain(state):
    case = state["case"]
    op = case["op"]
    if op == "route":
        return _plain_route(state["logits"], case["top_k"], case["scoring"], case["normalise"], case["scale"],
                            state["bias"])
    if op == "block":
        b = (state["weights"][:, :, None] * state["y"].float()).sum(dim=1)
        if state["post"] is not None:
            b = _plain_norm(b, state["post"], case["gemma"])
        if state["gate"] is not None:
            b = b * state["gate"].float()
        h = case["res_scale"] * state["h"].float() + b
        return h.to(torch.bfloat16), _plain_norm(h, state["next"], case["gemma"]).to(torch.bfloat16)
    ids = _plain_route(state["logits"], case["top_k"])[0]
    x = state["x"].float()
    if op == "grouped":
        w = state["w"]
        return _plain_by_expert(ids, case["experts"], case["n"],
                                lambda e, row: x[row] @ _plain_dense(*(t[e] for t in w)).T)

    def mlp(e, row):
        gate, up, down = (_plain_dense(*(t[e] for t in state[key])) for key in ("gate", "up", "down"))
        xe = x[row]
        return (_plain_act(xe @ gate.T, case["act"]) * (xe @ up.T)) @ down.T

    return _plain_by_expert(ids, case["experts"], case["hidden"], mlp)


# ---- the framework's operators ----------------------------------------------------------------------------------
def _own(state):
    from ironmule_b200 import kernels

    case = state["case"]
    op = case["op"]
    if op == "route":
        r = kernels.moe_route(state["logits"], case["top_k"], scoring=case["scoring"], normalise=case["normalise"],
                              scale=case["scale"], bias=state["bias"])
        return r.ids, r.weights, r.offsets, r.pairs
    if op == "block":
        return kernels.block_residual(state["y"], state["h"], EPS, weights=state["weights"], post_norm=state["post"],
                                      gate=state["gate"], residual_scale=case["res_scale"], next_norm=state["next"],
                                      gemma=case["gemma"])
    routing = kernels.moe_route(state["logits"], case["top_k"])
    if op == "grouped":
        return kernels.grouped_qgemm(state["x"], state["packed"], routing)
    return kernels.moe_mlp(state["x"], *state["packed"], routing, activation=case["act"])


def run(state):
    return _own(state) if own else _plain(state)


# ---- exact values -----------------------------------------------------------------------------------------------
def _exact_ids(logits, top_k, bias=None):
    """Per row, the k largest 32-bit keys (ties to the lower expert), -1 where fewer are open; numpy on the host."""
    import numpy as np

    values = logits.float().cpu().numpy()
    keys = values if bias is None else values + bias.cpu().numpy()
    order = np.argsort(-keys, axis=1, kind="stable")[:, :top_k]
    return np.where(np.isneginf(np.take_along_axis(values, order, 1)), -1, order)


def _exact_matrix(w, scales, biases):
    nibbles = torch.stack([(w >> (4 * i)) & 15 for i in range(8)], dim=2).flatten(1).double()
    return nibbles * scales.double().repeat_interleave(GROUP, 1) + biases.double().repeat_interleave(GROUP, 1)


def exact(case, seed):
    import numpy as np

    state = _inputs(case, seed)
    op = case["op"]
    if op == "block":
        out = torch.zeros((case["rows"], case["hidden"]), dtype=torch.float64, device="cuda")
        for j in range(case["places"]):
            out += state["weights"][:, j, None].double() * state["y"][:, j].double()

        def norm(v, w):
            rms = torch.rsqrt(v.square().sum(1, keepdim=True) / case["hidden"] + EPS)
            return rms * v * (w.double() + (1.0 if case["gemma"] else 0.0))

        if case["post"]:
            out = norm(out, state["post"])
        if state["gate"] is not None:
            out = out * state["gate"].double()
        out = out + state["h"].double() * case["res_scale"]
        return out, norm(out, state["next"])
    if op == "route":
        ids = _exact_ids(state["logits"], case["top_k"], state["bias"])
        values = state["logits"].double().cpu().numpy()
        live = ids >= 0
        picked = np.take_along_axis(values, np.maximum(ids, 0), 1)
        if case["scoring"] == "softmax":
            top = values.max(axis=1, keepdims=True)
            top = np.where(np.isneginf(top), 0.0, top)
            scores, every = np.exp(picked - top), np.exp(values - top).sum(axis=1, keepdims=True)
        else:
            scores, every = np.reciprocal(1.0 + np.exp(-picked)), 1.0
        scores = np.where(live, scores, 0.0)
        if case["normalise"]:
            every = scores.sum(axis=1, keepdims=True)
        weights = np.divide(scores * case["scale"], every, out=np.zeros_like(scores), where=live)
        bucket = np.where(live, ids, case["experts"]).ravel()
        offsets = np.concatenate([[0], np.cumsum(np.bincount(bucket, minlength=case["experts"] + 1))])
        return (torch.from_numpy(ids.astype(np.int32)), torch.from_numpy(weights),
                torch.from_numpy(offsets.astype(np.int32)),
                torch.from_numpy(np.argsort(bucket, kind="stable").astype(np.int32)))
    ids = torch.from_numpy(_exact_ids(state["logits"], case["top_k"])).to("cuda")
    x = state["x"].double()
    width = case["n"] if op == "grouped" else case["hidden"]
    y = torch.zeros((*ids.shape, width), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        row, place = torch.nonzero(ids == e, as_tuple=True)
        if not row.numel():
            continue
        if op == "grouped":
            y[row, place] = torch.matmul(x[row], _exact_matrix(*(t[e] for t in state["w"])).t())
            continue
        g = torch.matmul(x[row], _exact_matrix(*(t[e] for t in state["gate"])).t())
        u = torch.matmul(x[row], _exact_matrix(*(t[e] for t in state["up"])).t())
        if case["act"] == "swiglu":
            a = g * torch.sigmoid(g)
        else:
            a = g * 0.5 * (torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g**3)) + 1.0)
        y[row, place] = torch.matmul(a * u, _exact_matrix(*(t[e] for t in state["down"])).t())
    return y


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def _chosen(case):
    """Experts that some row chose, on average, were every choice equally likely."""
    return case["experts"] * (1.0 - (1.0 - case["top_k"] / case["experts"]) ** case["rows"])


def work(case):
    op, rows = case["op"], case["rows"]
    if op == "block":
        hidden, gate = case["hidden"], {"none": 0, "channel": case["hidden"], "row": rows, "full": rows * case["hidden"]}
        vectors = (2 if case["post"] else 1) * hidden + gate[case["gate"]]
        return {"bytes": 2 * (rows * case["places"] * hidden + 3 * rows * hidden + vectors) + 4 * rows * case["places"],
                "flops": rows * hidden * (2 * case["places"] + 10)}
    pairs = rows * case["top_k"]
    logits = rows * case["experts"] * (4 if case.get("dtype") == "f32" else 2)
    if op == "route":
        return {"bytes": logits + 4 * (3 * pairs + case["experts"] + 2 + (case["experts"] if case["bias"] else 0)),
                "flops": 4 * rows * case["experts"]}
    live = pairs * (0.875 if case.get("closed") else 1.0)
    if op == "grouped":
        weights, width = case["n"] * case["k"], case["n"]
        read = rows * case["k"]
    else:
        weights, width = 3 * case["hidden"] * case["inter"], case["hidden"]
        read = rows * case["hidden"]
    return {"bytes": int(_chosen(case) * weights * 9 / 16) + logits + 2 * (read + pairs * width),
            "flops": int(2 * live * weights)}
