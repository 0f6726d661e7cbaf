"""What decoding over a bounded cache is measured on: cases, inputs, the operators' plain form and their exact values.

Five operators over a cache of 16-slot pages, [pages, Hkv, 16, D]:

  rope_kv  packed q, k, v rows: q and k rotated to their positions; k, v and the position written to the cache
  rope     rows rotated to their positions, or back (which is the rotation's gradient)
  attend   rows attend to their sequence's slots, and every slot's weight is added to what it had
  evict    of each kv head's slots a budget stays: the newest, the first, the heaviest; the cache is closed up
  verify   drafted tokens kept or refused from probabilities and given random numbers, then one more token drawn

`run` computes them with elementary torch operations, or, where `own` is true, through ironmule_b200.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ---- cases ----------------------------------------------------------------------------------------------------
def _rope_kv(name, rows, seqs, hq, hkv, d, rotary, layout="half", dtype="bf16", table="plain", start=0, shift=0, pad=0):
    return {"name": name, "op": "rope_kv", "rows": rows, "seqs": seqs, "hq": hq, "hkv": hkv, "d": d, "rotary": rotary,
            "layout": layout, "dtype": dtype, "table": table, "start": start, "shift": shift, "pad": pad}


def _rope(name, rows, heads, d, rotary, layout, dtype, table="plain", far=4096, inverse=False):
    return {"name": name, "op": "rope", "rows": rows, "heads": heads, "d": d, "rotary": rotary, "layout": layout,
            "dtype": dtype, "table": table, "far": far, "inverse": inverse}


def _attend(name, seqs, rows, slots, hq, hkv, d, dtype="bf16", window=0, ragged=True, idle=0):
    return {"name": name, "op": "attend", "seqs": seqs, "rows": rows, "slots": slots, "hq": hq, "hkv": hkv, "d": d,
            "dtype": dtype, "window": window, "ragged": ragged, "idle": idle}


def _evict(name, layers, seqs, slots, budget, recent, sinks, hkv, d, dtype="bf16", before=False, ragged=False):
    return {"name": name, "op": "evict", "layers": layers, "seqs": seqs, "slots": slots, "budget": budget,
            "recent": recent, "sinks": sinks, "hkv": hkv, "d": d, "dtype": dtype, "before": before, "ragged": ragged}


def _verify(name, seqs, drafts, vocab, dtype="f32", dist=True, ragged=False):
    return {"name": name, "op": "verify", "seqs": seqs, "drafts": drafts, "vocab": vocab, "dtype": dtype, "dist": dist,
            "ragged": ragged}


def listed():
    return [
        # one decoded token of a long text whose cache was cut down: position and slot differ
        _rope_kv("rope-token", 1, 1, 32, 8, 128, 128, start=2047, shift=98000),
        # a prompt's prefill in one piece, frequencies stretched for a long context
        _rope_kv("rope-prompt", 8192, 1, 32, 8, 128, 128, table="yarn"),
        # the rotation's gradient at odd sizes: float32, neighbouring pairs, part of the head, far positions
        _rope("rope-gradient", 2049, 20, 96, 48, "interleaved", "f32", table="linear", far=2**20, inverse=True),
        # one decoded token: latency is everything
        _attend("attend-token", 1, 1, 2048, 32, 8, 128, ragged=False),
        # one decoded token of 32 sequences of different lengths
        _attend("attend-batch", 32, 1, 8192, 32, 8, 128),
        # a verification pass over a sliding window: four drafts and the last token, wide heads, two idle sequences
        _attend("attend-verify", 8, 5, 4001, 16, 8, 256, window=1024, idle=2),
        # one sequence over a very long cache of an odd length
        _attend("attend-long", 1, 1, 131071, 32, 8, 128, ragged=False),
        # one page's worth of new tokens evicted from a full cache, every layer at once
        _evict("evict-step", 36, 1, 2064, 2048, 256, 4, 8, 128, before=True),
        # a prompt's cache cut to a quarter, every layer at once
        _evict("evict-prompt", 36, 1, 8192, 2048, 256, 4, 8, 128),
        # sequences of odd lengths, some within the budget already, one layer
        _evict("evict-batch", 13, 12, 1777, 1000, 33, 0, 4, 64, dtype="f16", ragged=True),
        # one sequence's four drafts
        _verify("verify-token", 1, 4, 151936),
        # 32 sequences of up to four drafts each
        _verify("verify-batch", 32, 4, 151936, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope_kv", "rope", "attend", "attend", "evict", "verify"])
    if op in ("rope_kv", "rope"):
        d = 16 * rng.randint(2, 16)
        rotary = rng.choice([d, d, d // 2, 16 * rng.randint(1, d // 16)])
        layout, table = rng.choice(["half", "interleaved"]), rng.choice(["plain", "linear", "yarn"])
        if op == "rope_kv":
            hkv = rng.choice([1, 2, 3, 4, 8])
            hq = hkv * rng.choice([1, 2, 4, 5])
            most = 8192 * 48 * 128 // ((hq + 2 * hkv) * d)
            rows = _log_int(rng, 1, min(8192, most))
            seqs = rng.randint(1, min(rows, 32))
            return _strip(_rope_kv("", rows, seqs, hq, hkv, d, rotary, layout, rng.choice(["bf16", "f16"]), table,
                                   rng.randint(0, 500), rng.choice([0, _log_int(rng, 1, 2**20)]),
                                   rng.choice([0, 0, rows // 5])))
        heads, dtype = rng.randint(1, 40), rng.choice(["bf16", "f16", "f32"])
        rows = _log_int(rng, 1, min(8192, 8192 * 48 * 128 // (heads * d * (2 if dtype == "f32" else 1))))
        return _strip(_rope("", rows, heads, d, rotary, layout, dtype, table, _log_int(rng, 64, 2**20),
                            rng.random() < 0.5))
    dtype = rng.choice(["bf16", "f16"])
    d = rng.choice([64, 80, 96, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 5, 8])
    if op == "attend":
        seqs, rows = _log_int(rng, 1, 32), rng.choice([1, 1, 1, 2, 5, 9])
        hq = hkv * rng.choice([1, 2, 4, 7, 8])
        slots = _log_int(rng, 1, 131072)
        while seqs > 1 and seqs * slots * hkv * d > 16 * 8192 * 8 * 128:
            seqs //= 2
        while slots > 64 and seqs * slots * rows * hq * d > 16 * 8192 * 32 * 128:
            slots //= 2
        return _strip(_attend("", seqs, rows, max(slots, rows), hq, hkv, d, dtype, rng.choice([0, 0, 512]),
                              rng.random() < 0.7, rng.choice([0, 0, seqs // 3])))
    if op == "evict":
        layers, seqs, slots = _log_int(rng, 1, 36), _log_int(rng, 1, 16), _log_int(rng, 4, 65536)
        while seqs > 1 and layers * seqs * slots * hkv * d > 36 * 8192 * 8 * 128:
            seqs //= 2
        while layers > 1 and layers * slots * hkv * d > 36 * 8192 * 8 * 128:
            layers //= 2
        budget = rng.choice([slots // 4, slots // 2, slots - min(16, slots // 3)])
        recent, sinks = rng.choice([0, budget // 8, budget // 2]), rng.choice([0, min(4, budget // 2)])
        return _strip(_evict("", layers, seqs, slots, max(1, budget), recent, sinks, hkv, d, dtype, rng.random() < 0.5,
                             rng.random() < 0.5))
    vocab, seqs, drafts = _log_int(rng, 500, 262144), _log_int(rng, 1, 64), rng.randint(0, 8)
    while seqs > 1 and seqs * (drafts + 1) * vocab > 32 * 5 * 151936:
        seqs //= 2
    return _strip(_verify("", seqs, drafts, vocab, rng.choice(["f32", "f32", "bf16"]), rng.random() < 0.7,
                          rng.random() < 0.5))


def _strip(case):
    del case["name"]
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------
def _normal(gen, *shape, std=1.0, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype) * std


def _uniform(gen, *shape):
    return torch.rand(shape, generator=gen, device="cuda")


def _table(kind, rotary):
    """Angles per position of each pair (float64), and the factor on the rotated values."""
    base, i = 1_000_000.0, torch.arange(rotary // 2, dtype=torch.float64)
    freq = base ** (-2.0 * i / rotary)
    if kind == "plain":
        return freq.cuda(), 1.0
    if kind == "linear":
        return (freq / 8.0).cuda(), 1.0
    stretch, trained = 4.0, 32768

    def pair(turns):  # the pair that makes so many turns over the trained length
        return rotary * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(base))

    low, high = max(0, math.floor(pair(32.0))), min(rotary - 1, math.ceil(pair(1.0)))
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return (freq / stretch * ramp + freq * (1 - ramp)).cuda(), 0.1 * math.log(stretch) + 1.0


def _pages(gen, seqs, slots):
    """A page table of that many slots a sequence, its pages in no order, and their number."""
    per = -(-slots // PAGE)
    order = torch.argsort(_uniform(gen, seqs * per))
    return order.to(torch.int32).view(seqs, per).contiguous(), seqs * per


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    int32 = {"device": "cuda", "dtype": torch.int32}
    if op == "rope":
        freq, factor = _table(case["table"], case["rotary"])
        heads, d = case["heads"], case["d"]
        # the heads lie in a wider row, as they do in a packed projection
        packed = _normal(gen, case["rows"], (heads + 2) * d, dtype=torch.float32).to(dtype)
        return {"x": packed[:, : heads * d].view(case["rows"], heads, d), "freq": freq, "factor": factor,
                "pos": torch.randint(0, case["far"], (case["rows"],), generator=gen, **int32)}
    if op == "rope_kv":
        freq, factor = _table(case["table"], case["rotary"])
        rows, seqs, hkv, d = case["rows"], case["seqs"], case["hkv"], case["d"]
        live = max(1, rows - case["pad"])
        per = -(-live // seqs)
        row = torch.arange(rows, **int32)
        slots = case["start"] + per
        table, pages = _pages(gen, seqs, slots)
        slot = torch.where(row < live, case["start"] + row % per, -1).to(torch.int32)
        return {"qkv": _normal(gen, rows, (case["hq"] + 2 * hkv) * d).to(dtype), "freq": freq, "factor": factor,
                "pos": (slot.clamp(min=0) + case["shift"]).to(torch.int32), "slot": slot,
                "seq": (row // per).clamp(max=seqs - 1).to(torch.int32), "table": table,
                "k": torch.zeros((pages, hkv, PAGE, d), device="cuda", dtype=dtype),
                "v": torch.zeros((pages, hkv, PAGE, d), device="cuda", dtype=dtype),
                "slot_pos": torch.full((seqs, hkv, table.shape[1] * PAGE), -1, **int32)}
    if op == "attend":
        seqs, rows, slots, hkv, d = case["seqs"], case["rows"], case["slots"], case["hkv"], case["d"]
        table, pages = _pages(gen, seqs, slots)
        cap = table.shape[1] * PAGE
        length = torch.full((seqs,), slots, **int32)
        if case["ragged"]:
            length = (slots * (0.5 + 0.5 * _uniform(gen, seqs))).to(torch.int32).clamp(rows, slots)
        slot = length[:, None] - rows + torch.arange(rows, **int32)
        if case["idle"]:  # sequences without a token in this pass: their rows see nothing
            slot[torch.argsort(_uniform(gen, seqs))[: case["idle"]]] = -1
        k = torch.empty((pages, hkv, PAGE, d), device="cuda", dtype=dtype)
        k.normal_(generator=gen)
        k *= (0.5 + 2.0 * _uniform(gen, pages, hkv, PAGE, 1) ** 4).to(dtype)  # a few keys draw much of the weight
        v = torch.empty_like(k)
        v.normal_(generator=gen)
        return {"q": _normal(gen, seqs * rows, case["hq"], d).to(dtype), "k": k, "v": v, "table": table,
                "seq_rows": torch.arange(seqs + 1, **int32) * rows, "slot": slot.flatten().to(torch.int32).contiguous(),
                "before": 4.0 * _uniform(gen, seqs, hkv, cap) ** 8, "after": torch.zeros((seqs, hkv, cap), device="cuda"),
                "scale": d ** -0.5}
    if op == "evict":
        layers, seqs, slots, hkv, d = case["layers"], case["seqs"], case["slots"], case["hkv"], case["d"]
        table, pages = _pages(gen, seqs, slots)
        cap = table.shape[1] * PAGE
        length = torch.full((seqs,), slots, **int32)
        if case["ragged"]:
            length = (slots * _uniform(gen, seqs)).to(torch.int32).clamp(1, slots)
        k = torch.empty((layers, pages, hkv, PAGE, d), device="cuda", dtype=dtype)
        k.normal_(generator=gen)
        v = torch.empty_like(k)
        v.normal_(generator=gen)
        # sums of attention weights: most small, a few large, some slots never looked at
        weights = torch.exp(_normal(gen, layers, seqs, hkv, cap, std=1.5))
        weights = weights * (_uniform(gen, layers, seqs, hkv, cap) > 0.1)
        pos = torch.arange(cap, **int32).expand(layers, seqs, hkv, cap)
        seen = length.clone()
        if case["before"]:  # earlier evictions left the older slots in no order, and gaps in their positions
            seen = 3 * length
            new = min(PAGE, slots // 3)
            old = 3 * torch.argsort(_uniform(gen, layers, seqs, hkv, cap), dim=-1).to(torch.int32)
            newest = (torch.arange(cap, **int32) - length[:, None] + seen[:, None])[None, :, None, :]
            fresh = (torch.arange(cap, **int32) >= length[:, None] - new)[None, :, None, :]
            pos = torch.where(fresh, newest, torch.minimum(old, (seen[:, None] - new - 1).clamp(min=0)[None, :, None, :]))
        return {"k": k, "v": v, "table": table, "length": length, "seen": seen.to(torch.int32), "weights": weights,
                "pos": pos.to(torch.int32).contiguous(), "weights_out": torch.zeros_like(weights),
                "pos_out": torch.full((layers, seqs, hkv, cap), -1, **int32)}
    seqs, drafts, vocab = case["seqs"], case["drafts"], case["vocab"]
    logits = _normal(gen, seqs, drafts + 1, vocab, std=3.0)
    near = logits[:, :drafts] + _normal(gen, seqs, drafts, vocab, std=0.7)

    def filtered(x):  # as after a top-p filter: small probabilities are zero
        x = torch.softmax(x, dim=-1)
        x = torch.where(x >= 1e-3 * x.amax(dim=-1, keepdim=True), x, 0.0)
        return (x / x.sum(dim=-1, keepdim=True)).to(dtype)

    p = filtered(logits)
    q = filtered(near) if drafts else torch.zeros((seqs, 0, vocab), device="cuda", dtype=dtype)
    state = {"p": p, "q": q if case["dist"] and drafts else None, "u": _uniform(gen, seqs, drafts + 1), "n": None}
    if drafts:
        picked = torch.multinomial(q.float().view(seqs * drafts, vocab), 1, generator=gen).view(seqs, drafts)
        state["drafts"] = picked.to(torch.int32)
    else:
        state["drafts"] = torch.zeros((seqs, 0), **int32)
    if case["ragged"]:
        state["n"] = torch.randint(0, drafts + 1, (seqs,), generator=gen, **int32)
    return state


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    return state


# ---- the plain form -------------------------------------------------------------------------------------------
def _plain_rotate(x, pos, freq, factor, layout, inverse=False):
    """x [M, H, D] in 32 bits; angles in 64, since positions are far."""
    angle = pos.double()[:, None] * freq
    cos, sin = ((factor * f(angle)).float()[:, None] for f in (torch.cos, torch.sin))
    sin = -sin if inverse else sin
    rotary = 2 * freq.numel()
    if layout == "half":
        a, b = x[..., : rotary // 2], x[..., rotary // 2 : rotary]
        turned = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    else:
        a, b = x[..., 0:rotary:2], x[..., 1:rotary:2]
        turned = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    return torch.cat([turned, x[..., rotary:]], dim=-1)


def _plain_rope_kv(state, case):
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    qkv = state["qkv"].view(-1, hq + 2 * hkv, d)
    turned = _plain_rotate(qkv[:, : hq + hkv].float(), state["pos"], state["freq"], state["factor"], case["layout"])
    turned = turned.to(qkv.dtype)
    live = (state["slot"] >= 0).nonzero()[:, 0]
    slot, seq = state["slot"][live].long(), state["seq"][live].long()
    page = state["table"][seq, slot // PAGE].long()
    state["k"][page, :, slot % PAGE] = turned[live, hq:]
    state["v"][page, :, slot % PAGE] = qkv[live, hq + hkv :]
    state["slot_pos"][seq, :, slot] = state["pos"][live][:, None].expand(-1, hkv)
    return turned[:, :hq].contiguous(), state["k"], state["v"], state["slot_pos"]


def _plain_attend(state, case):
    seqs, rows, hkv, d = case["seqs"], case["rows"], case["hkv"], case["d"]
    group = case["hq"] // hkv
    table = state["table"].long()
    cap = table.shape[1] * PAGE
    slot = state["slot"].view(seqs, rows)
    key = torch.arange(cap, device="cuda")
    seen = key <= slot[:, :, None]
    if case["window"]:
        seen &= key > slot[:, :, None] - case["window"]
    k = state["k"][table].transpose(1, 2).reshape(seqs, hkv, cap, d).float()
    q = state["q"].view(seqs, rows, hkv, group, d).permute(0, 2, 1, 3, 4).reshape(seqs, hkv, rows * group, d).float()
    s = state["scale"] * (q @ k.transpose(-1, -2)).view(seqs, hkv, rows, group, cap)
    del k
    s = s.masked_fill(~seen[:, None, :, None], float("-inf"))
    top = s.amax(dim=-1, keepdim=True)
    p = torch.exp(s - torch.where(top > float("-inf"), top, 0.0))
    p = p / p.sum(dim=-1, keepdim=True).clamp(min=1e-30)
    used = key <= slot[:, -1:]
    v = state["v"][table].transpose(1, 2).reshape(seqs, hkv, cap, d).float()
    v = v.masked_fill(~used[:, None, :, None], 0.0)
    out = (p.view(seqs, hkv, rows * group, cap) @ v).view(seqs, hkv, rows, group, d)
    old = torch.where((key < slot[:, :1])[:, None], state["before"], 0.0)
    state["after"].copy_(torch.where(used[:, None], old + p.sum(dim=(2, 3)), state["after"]))
    out = out.permute(0, 2, 1, 3, 4).reshape(seqs * rows, case["hq"], d)
    return out.to(state["q"].dtype), state["after"]


def _plain_evict(state, case):
    cap = state["weights"].shape[-1]
    slot = torch.arange(cap, device="cuda")
    length = state["length"][None, :, None, None]
    left = length.clamp(max=case["budget"])
    pos, weights = state["pos"], state["weights"]
    valid = slot < length
    safe = (pos < case["sinks"]) | (pos >= state["seen"][None, :, None, None] - case["recent"])
    key = torch.where(safe, float("inf"), weights).masked_fill(~valid, float("-inf"))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, slot.expand_as(order).contiguous())
    kept = rank < left
    # the i-th kept slot behind the new end goes to the i-th dropped slot before it
    hole, mover = (valid & (slot < left) & ~kept).nonzero(as_tuple=True), (kept & (slot >= left)).nonzero(as_tuple=True)
    before = slot < left
    state["weights_out"].copy_(torch.where(before, weights, state["weights_out"]))
    state["pos_out"].copy_(torch.where(before, pos, state["pos_out"]))
    state["weights_out"][hole], state["pos_out"][hole] = weights[mover], pos[mover]
    table = state["table"].long()
    to, source = ((at[0], table[at[1], at[3] // PAGE], at[2], at[3] % PAGE) for at in (hole, mover))
    state["k"][to], state["v"][to] = state["k"][source], state["v"][source]
    return left.flatten().to(torch.int32), state["weights_out"], state["pos_out"], state["k"], state["v"]


def _plain_verify(state, case):
    """In 64 bits: a drawn token lies next to a border of the cumulative sum."""
    seqs, drafts = state["drafts"].shape
    p, u = state["p"], state["u"].double()
    place = torch.arange(drafts, device="cuda")
    count = torch.full((seqs,), drafts, device="cuda") if state["n"] is None else state["n"].long()
    if drafts:
        token = state["drafts"].long()[..., None]
        chance = torch.gather(p[:, :drafts], 2, token)[..., 0].double()
        offered = 1.0 if state["q"] is None else torch.gather(state["q"], 2, token)[..., 0].double()
        good = (u[:, :drafts] * offered < chance) & (place < count[:, None])
        kept = torch.cumprod(good.long(), dim=1).sum(dim=1)
    else:
        kept = torch.zeros(seqs, device="cuda", dtype=torch.int64)
    every = torch.arange(seqs, device="cuda")
    weight = p[every, kept].double()
    if drafts:
        refused, at = (kept < count)[:, None], kept.clamp(max=drafts - 1)
        if state["q"] is None:
            less = weight.scatter(1, state["drafts"][every, at].long()[:, None], 0.0)
        else:
            less = (weight - state["q"][every, at].double()).clamp(min=0.0)
        less = torch.where(refused, less, weight)
        weight = torch.where(less.sum(dim=1, keepdim=True) > 0, less, weight)
    total = torch.cumsum(weight, dim=1)
    last = torch.gather(u, 1, torch.full((seqs, 1), drafts, device="cuda"))
    drawn = (total > last * total[:, -1:]).to(torch.int32).argmax(dim=1)
    step = torch.arange(drafts + 1, device="cuda")
    tokens = torch.full((seqs, drafts + 1), -1, device="cuda", dtype=torch.int64)
    tokens[:, :drafts] = torch.where(place < kept[:, None], state["drafts"].long(), -1)
    tokens = torch.where(step == kept[:, None], drawn[:, None], tokens)
    return tokens.to(torch.int32), (kept + 1).to(torch.int32)


def _plain(state):
    case = state["case"]
    if case["op"] == "rope":
        return _plain_rotate(state["x"].float(), state["pos"], state["freq"], state["factor"], case["layout"],
                             case["inverse"]).to(state["x"].dtype)
    return {"rope_kv": _plain_rope_kv, "attend": _plain_attend, "evict": _plain_evict,
            "verify": _plain_verify}[case["op"]](state, case)


# ---- the framework's operators ----------------------------------------------------------------------------------
def _own(state):
    from ironmule_b200 import kernels

    case = state["case"]
    op = case["op"]
    if op == "rope":
        return kernels.rope(state["x"], state["pos"], state["freq"], layout=case["layout"], factor=state["factor"],
                            inverse=case["inverse"])
    if op == "rope_kv":
        q = kernels.rope_kv(state["qkv"], state["freq"], state["pos"], state["slot"], state["seq"], state["table"],
                            case["hq"], case["hkv"], case["d"], state["k"], state["v"], layout=case["layout"],
                            factor=state["factor"], slot_pos=state["slot_pos"])
        return q, state["k"], state["v"], state["slot_pos"]
    if op == "attend":
        out = kernels.attention_weights(state["q"], state["k"], state["v"], state["table"], state["seq_rows"],
                                        state["slot"], state["before"], max_rows_per_seq=case["rows"],
                                        max_kv_len=case["slots"], scale=state["scale"], window=case["window"],
                                        weights_out=state["after"])
        return out, state["after"]
    if op == "evict":
        left = kernels.cache_evict(state["k"], state["v"], state["table"], state["length"], state["seen"],
                                   state["weights"], state["pos"], budget=case["budget"], recent=case["recent"],
                                   sinks=case["sinks"], weights_out=state["weights_out"], pos_out=state["pos_out"])
        return left, state["weights_out"], state["pos_out"], state["k"], state["v"]
    return kernels.verify_sampled(state["p"], state["q"], state["drafts"], state["u"], n_drafts=state["n"])


def run(state):
    return _own(state) if own else _plain(state)


# ---- exact values -----------------------------------------------------------------------------------------------
def _exact_turn(x, pos, freq, factor, layout, back):
    """Each pair as a complex number times factor e^(it)."""
    t = pos.double()[:, None, None] * freq.double()
    turn = torch.polar(torch.full_like(t, factor), -t if back else t)
    x, rotary = x.double(), 2 * freq.numel()
    head = x[..., :rotary]
    pairs = head.unflatten(-1, (2, rotary // 2)).transpose(-1, -2) if layout == "half" else head.unflatten(-1, (-1, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn)
    head = (z.transpose(-1, -2) if layout == "half" else z).flatten(-2)
    return torch.cat([head, x[..., rotary:]], dim=-1)


def exact(case, seed):
    state, op = _inputs(case, seed), case["op"]
    if op == "rope":
        return _exact_turn(state["x"], state["pos"], state["freq"], state["factor"], case["layout"], case["inverse"])
    if op == "rope_kv":
        hq, hkv = case["hq"], case["hkv"]
        qkv = state["qkv"].view(case["rows"], hq + 2 * hkv, case["d"])
        turned = _exact_turn(qkv[:, : hq + hkv], state["pos"], state["freq"], state["factor"], case["layout"], False)
        k, v = state["k"].double(), state["v"].double()
        on = state["slot"] >= 0
        slot, seq = state["slot"][on].long(), state["seq"][on].long()
        at = state["table"][seq, slot.div(PAGE, rounding_mode="floor")].long()
        k[at, :, slot.remainder(PAGE)] = turned[on, hq:]
        v[at, :, slot.remainder(PAGE)] = qkv[on, hq + hkv :].double()
        return turned[:, :hq], k, v, None
    if op != "attend":
        return None  # whole numbers, and values that are moved as they are
    out, after = torch.zeros_like(state["q"], dtype=torch.float64), state["after"].double()
    group = case["hq"] // case["hkv"]
    for b in range(case["seqs"]):
        rows = slice(b * case["rows"], (b + 1) * case["rows"])
        slots = state["slot"][rows].tolist()
        if slots[-1] < 0:
            continue
        n = slots[-1] + 1
        pages = state["table"][b, : -(-n // PAGE)].long()
        for h in range(case["hkv"]):
            k, v = (state[t][pages, h].flatten(0, 1)[:n].double() for t in ("k", "v"))
            after[b, h, : slots[0]] = state["before"][b, h, : slots[0]].double()
            for r, last in enumerate(slots):
                first = max(0, last + 1 - case["window"]) if case["window"] else 0
                heads = slice(h * group, (h + 1) * group)
                qs = state["q"][rows][r, heads].double() * state["scale"]
                p = torch.softmax(k[first : last + 1] @ qs.T, dim=0)
                out[rows][r, heads] = p.T @ v[first : last + 1]
                after[b, h, first : last + 1] += p.sum(dim=1)
    return out, after


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    op, size = case["op"], 4 if case["dtype"] == "f32" else 2
    if op == "rope":
        values = case["rows"] * case["heads"] * case["d"]
        return {"bytes": 2 * size * values + 4 * case["rows"], "flops": 3 * values * case["rotary"] // case["d"]}
    if op == "rope_kv":
        hq, hkv, d = case["hq"], case["hkv"], case["d"]
        live = max(1, case["rows"] - case["pad"])
        return {"bytes": size * d * (2 * case["rows"] * hq + 4 * live * hkv) + 12 * case["rows"] + 4 * live * hkv,
                "flops": 3 * case["rows"] * (hq + hkv) * case["rotary"]}
    if op == "attend":
        live = case["seqs"] - case["idle"]
        length = live * (case["slots"] * (0.75 if case["ragged"] else 1.0))
        seen = min(length, live * (case["window"] + case["rows"])) if case["window"] else length
        rows = case["seqs"] * case["rows"] * case["hq"] * case["d"]
        return {"bytes": int(seen * case["hkv"] * 2 * size * case["d"] + 8 * length * case["hkv"] + 2 * size * rows),
                "flops": int(4 * seen * case["rows"] * case["hq"] * case["d"])}
    if op == "evict":
        heads = case["layers"] * case["seqs"] * case["hkv"]
        share = 0.5 if case["ragged"] else 1.0
        left = min(case["budget"], case["slots"] * share)
        over = max(0.0, case["slots"] - case["budget"]) / case["slots"] * share
        free = max(0, case["budget"] - case["recent"])
        moved = over * (case["recent"] + free * over) if not case["before"] else over * case["budget"]
        return {"bytes": int(heads * (8 * case["slots"] * share + 8 * left + 4 * size * case["d"] * moved)),
                "flops": int(heads * case["slots"] * share)}
    rows = case["seqs"] * case["vocab"] * (2 if case["dist"] and case["drafts"] else 1)
    return {"bytes": size * rows + 4 * case["seqs"] * 3 * (case["drafts"] + 1), "flops": 3 * rows}
