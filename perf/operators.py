"""Operators of wide decoding -- many requests a step -- in cases that can be timed and checked.

A step reads its weights once for all of its requests, and every request's cache.  Three operators make both smaller:

* ``linear``: a matrix product in 8-bit integers.  Every token's row and every channel's weights are brought to
  integers of [-127, 127] by a scale of their own, ``scale = max|x| / 127`` rounded to 32 bits and
  ``value = round(x / scale)`` (ties to even); the integer sums are exact, and both scales go on behind them.  With a
  residual row added behind the scales, or rounded to bfloat16.
* ``gated``: the gated feed-forward's first half on the same integers: an RMS norm whose rows leave as integers, gate and
  up projection, ``act(gate) * up``.
* ``shared``: attention of requests whose first pages are the same ones (a system prompt, one prompt's many answers):
  every group's shared keys and values are read once for the whole group, every request's own ones behind them.

``own`` False: the plain forms, elementary torch in 32 bits (64 for the integer sums and for what decides a rounding).
``exact``: the definitions in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False
DEVICE = "cuda:0"
PAGE = 64


# ------------------------------------------------------------------ the cases
def _linear(name, tokens, inner, features, x="bfloat16", out="float32", residual=True):
    return {"name": name, "kind": "linear", "tokens": tokens, "inner": inner, "features": features, "x": x, "out": out,
            "residual": residual}


def _gated(name, tokens, inner, features, act="silu"):
    return {"name": name, "kind": "gated", "tokens": tokens, "inner": inner, "features": features, "act": act}


def _shared(name, groups, requests, tokens, prefix, own_keys, heads, kv_heads, dim, dtype="bfloat16", sink=False,
            softcap=0.0, idle=0):
    """``groups`` groups of up to ``requests`` requests with ``tokens`` tokens each behind up to ``prefix`` shared and
    ``own_keys`` own keys; ``idle`` rows of a padded batch behind the last group."""
    return {"name": name, "kind": "shared", "groups": groups, "requests": requests, "tokens": tokens, "prefix": prefix,
            "own_keys": own_keys, "heads": heads, "kv_heads": kv_heads, "dim": dim, "dtype": dtype, "sink": sink,
            "softcap": softcap, "idle": idle}


def listed():
    return [
        # one request's token through an output projection, into its residual row: latency alone
        _linear("linear-1x2048x2048", 1, 2048, 2048),
        # 64 decoding requests through the down projection: the weights' bytes
        _linear("linear-64x8192x2048", 64, 8192, 2048),
        # sizes that fill no tile, rows in 32 bits: a draft of a few hundred tokens in a model of odd width
        _linear("linear-333x1500x2047", 333, 1500, 2047, x="float32", out="bfloat16", residual=False),
        # a long prompt through the down projection: the tensor cores
        _linear("linear-4096x8192x2048", 4096, 8192, 2048),
        # eight decoding requests' gate and up projection behind their norm
        _gated("gated-8x2048x8192", 8, 2048, 8192),
        # a short prompt in a small model
        _gated("gated-200x1024x4608", 200, 1024, 4608, act="gelu_tanh"),
        # several prompts together
        _gated("gated-8192x2048x8192", 8192, 2048, 8192),
        # two answers to one short prompt
        _shared("shared-1x2-448", 1, 2, 1, 448, 60, 16, 8, 64),
        # 64 requests behind one system prompt, each with a turn of its own
        _shared("shared-1x64-8192", 1, 64, 1, 8192, 500, 32, 8, 64),
        # six applications' system prompts, three drafted tokens a request, a sink, rows of padding behind them
        _shared("shared-6x16-4096-sink", 6, 16, 3, 4096, 700, 24, 4, 128, sink=True, idle=7),
        # the 32-bit path with capped scores and a head size that is no power of two
        _shared("shared-2x10-1024-f32", 2, 10, 1, 1024, 130, 10, 5, 80, dtype="float32", softcap=20.0),
        # 256 requests over one long document
        _shared("shared-1x256-32768", 1, 256, 1, 32768, 1000, 32, 8, 64),
    ]


def _between(rng, low, high):
    """A whole number whose logarithm is spread evenly; half of them odd ones as they fall, half multiples of 64."""
    value = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if value > 256 and rng.random() < 0.5:
        value -= value % 64
    return max(low, min(high, value))


def draw(rng):
    kind = rng.choice(("linear", "gated", "shared", "shared"))
    if kind == "linear":
        residual = rng.random() < 0.5
        return _linear(None, _between(rng, 1, 4096), _between(rng, 64, 8192), _between(rng, 64, 8192),
                       x=rng.choice(("bfloat16", "float32")), out="float32" if residual else "bfloat16", residual=residual)
    if kind == "gated":
        return _gated(None, _between(rng, 1, 4096), _between(rng, 64, 4096), _between(rng, 64, 8192),
                      act=rng.choice(("silu", "gelu_tanh", "relu")))
    dtype = "float32" if rng.random() < 0.25 else "bfloat16"
    kv_heads = rng.choice((1, 2, 4, 5, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4, 8))
    dim = rng.choice((64, 64, 128, 128, 48, 96)) if dtype == "bfloat16" else rng.choice((32, 64, 80, 128))
    groups = rng.choice((1, 1, 2, 5))
    small = dtype == "float32" or dim not in (64, 128)
    case = _shared(None, groups, _between(rng, 1, 16 if small else 256), rng.choice((1, 1, 2, 4)),
                   _between(rng, 64, 2048 if small else 32768), _between(rng, 1, 300 if small else 1000), heads, kv_heads,
                   dim, dtype=dtype, sink=rng.random() < 0.3, softcap=20.0 if rng.random() < 0.2 else 0.0,
                   idle=rng.choice((0, 0, 5)))
    most = work(listed()[-1])["flops"]
    while work(case)["flops"] > most:                # no more than the largest listed one
        if case["requests"] > 1:
            case["requests"] //= 2
        else:
            case["prefix"] //= 2
    return case


# ------------------------------------------------------------------ the batch of a shared case, from the case alone
def _ragged(case):
    """Requests and shared pages of every group, own keys of every request.  The first group and the first request are
    the largest; the others fall off in steps."""
    requests = [max(1, case["requests"] - (g * 5) % case["requests"]) for g in range(case["groups"])]
    pages = [max(1, (case["prefix"] // PAGE) * (case["groups"] - g) // case["groups"]) for g in range(case["groups"])]
    most, least = case["own_keys"], min(case["tokens"], case["own_keys"])
    lengths = [max(least, most - (r * 37) % most) for r in range(sum(requests))]
    return requests, pages, lengths


def _counts(case):
    """(keys read once, (query, key) pairs, tokens) of a shared case."""
    requests, pages, lengths = _ragged(case)
    tokens = case["tokens"]
    read = PAGE * sum(pages) + sum(max(n, tokens) for n in lengths)
    pairs, r = 0, 0
    for count, shared in zip(requests, pages):
        for _ in range(count):
            n = max(lengths[r], tokens)
            pairs += sum(PAGE * shared + n - tokens + t + 1 for t in range(tokens))
            r += 1
    return read, pairs, tokens * sum(requests)


def work(case):
    if case["kind"] == "shared":
        size = 4 if case["dtype"] == "float32" else 2
        read, pairs, tokens = _counts(case)
        row = case["heads"] * case["dim"]
        return {"bytes": 2 * read * case["kv_heads"] * case["dim"] * size + 2 * tokens * row * size,
                "flops": 4 * pairs * row}
    m, k, n = case["tokens"], case["inner"], case["features"]
    if case["kind"] == "linear":
        out = 4 if case["out"] == "float32" else 2
        moved = m * k * (4 if case["x"] == "float32" else 2) + n * (k + 4) + m * n * (out + (4 if case["residual"] else 0))
        return {"bytes": moved, "flops": 2 * m * k * n}
    return {"bytes": 4 * m * k + 4 * k + 2 * n * (k + 4) + 2 * m * n, "flops": 4 * m * k * n}


# ------------------------------------------------------------------ inputs
def _quantized(x):
    """Rows of integers (as 64-bit floats) and their scales: max|x| / 127 rounded to 32 bits, round(x / scale)."""
    wide = x.double()
    scales = (wide.abs().amax(dim=-1) / 127.0).float()
    values = torch.where(scales[:, None] > 0, wide / scales.double()[:, None], torch.zeros_like(wide))
    return values.round().clamp(-127, 127), scales


def _activations(gen, rows, columns, dtype):
    """Rows with a few channels far larger than the others, as a transformer's are, and tokens of unequal size."""
    x = torch.randn(rows, columns, device=DEVICE, generator=gen)
    loud = torch.rand(columns, device=DEVICE, generator=gen) < 0.01
    x *= torch.where(loud, 6.0, 1.0)
    x *= torch.exp(0.3 * torch.randn(rows, 1, device=DEVICE, generator=gen))
    return x.to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["kind"] == "shared":
        return _prepare_shared(case, gen)
    m, k, n = case["tokens"], case["inner"], case["features"]
    rows = 2 * n if case["kind"] == "gated" else n
    weight = (torch.randn(rows, k, device=DEVICE, generator=gen) * k ** -0.5).to(torch.bfloat16)
    state = {"case": case}
    if case["kind"] == "gated":
        state["x"] = _activations(gen, m, k, torch.float32)
        state["norm"] = 1.0 + 0.1 * torch.randn(k, device=DEVICE, generator=gen)
    else:
        state["x"] = _activations(gen, m, k, getattr(torch, case["x"]))
        if case["residual"]:
            state["residual"] = torch.randn(m, n, device=DEVICE, generator=gen)
    if own:
        from flyweight_b200.kernels import int8
        state["weight"] = int8.matrix_int8(weight)       # laid out once, as a model's weights are
    else:
        state["weight"] = _quantized(weight)
    return state


def _prepare_shared(case, gen):
    requests, pages, lengths = _ragged(case)
    tokens, segments = case["tokens"], sum(requests)
    dtype = getattr(torch, case["dtype"])
    lengths = [max(n, tokens) for n in lengths]
    own_pages = [-(-n // PAGE) for n in lengths]
    shared_of, starts = [], [0]
    for count, shared in zip(requests, pages):
        shared_of += [shared] * count
        starts.append(starts[-1] + count * tokens)
    total = sum(pages) + sum(own_pages)
    order = torch.randperm(total, device=DEVICE, generator=gen).tolist()     # pages lie in the pool in no order
    table = torch.full((segments, max(s + o for s, o in zip(shared_of, own_pages))), -1, dtype=torch.int32)
    at, r = 0, 0
    for count, shared in zip(requests, pages):
        front, at = order[at:at + shared], at + shared
        for _ in range(count):
            rest, at = order[at:at + own_pages[r]], at + own_pages[r]
            table[r, :shared + own_pages[r]] = torch.tensor(front + rest, dtype=torch.int32)
            r += 1
    positions = [s * PAGE + n - tokens + t for s, n in zip(shared_of, lengths) for t in range(tokens)]
    segment = [r for r in range(segments) for _ in range(tokens)]
    idle = case["idle"]

    def device(values):
        return torch.tensor(values, dtype=torch.int32, device=DEVICE)

    pool = (total, case["kv_heads"], PAGE, case["dim"])
    rows = len(positions) + idle
    state = {"case": case, "positions": device(positions + [0] * idle), "segment": device(segment + [0] * idle),
             "table": table.to(DEVICE), "starts": device(starts), "pages": device(pages),
             "k": torch.randn(pool, device=DEVICE, generator=gen, dtype=dtype),
             "v": torch.randn(pool, device=DEVICE, generator=gen, dtype=dtype),
             "q": (1.5 * torch.randn(rows, case["heads"] * case["dim"], device=DEVICE, generator=gen)).to(dtype),
             "out": torch.zeros(rows, case["heads"] * case["dim"], device=DEVICE, dtype=dtype),
             "sink": torch.randn(case["heads"], device=DEVICE, generator=gen) if case["sink"] else None,
             "scale": case["dim"] ** -0.5, "most_tokens": tokens * max(requests), "most_pages": max(pages),
             "most_own": PAGE * max(own_pages)}
    return state


# ------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if case["kind"] == "shared":
        return _own_shared(state) if own else _plain_shared(state)
    if case["kind"] == "linear":
        return _own_linear(state) if own else _plain_linear(state)
    return _own_gated(state) if own else _plain_gated(state)


def _own_linear(state):
    from flyweight_b200.kernels import int8
    return int8.linear_int8(state["x"], state["weight"], getattr(torch, state["case"]["out"]), addend=state.get("residual"))


def _own_gated(state):
    from flyweight_b200.kernels import int8
    rows = int8.rmsnorm_int8(state["x"], state["norm"], 1e-5)
    return int8.gated_int8(rows, state["weight"], activation=state["case"]["act"])


def _own_shared(state):
    from flyweight_b200.kernels import attention
    case = state["case"]
    return attention.shared_prefix_attention(
        state["q"], state["k"], state["v"], state["positions"], state["segment"], state["table"], state["starts"],
        state["pages"], case["heads"], state["scale"], sink=state["sink"], softcap=case["softcap"], out=state["out"],
        shared_pages=state["most_pages"], own_pages=state["most_own"] // PAGE)


def _plain_product(values, scales, weight):
    """Exact integer sums (64-bit floats hold them) with both scales behind them, in 32 bits."""
    return ((values @ weight[0].T) * scales.double()[:, None] * weight[1].double()[None, :]).float()


def _plain_linear(state):
    y = _plain_product(*_quantized(state["x"]), state["weight"])
    if "residual" in state:
        y = y + state["residual"]
    return y.to(getattr(torch, state["case"]["out"]))


def _act(name, g):
    if name == "silu":
        return g * torch.sigmoid(g)
    if name == "relu":
        return torch.clamp(g, min=0)
    return 0.5 * g * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)))


def _plain_gated(state):
    wide = state["x"].double()              # what the norm gives decides roundings
    normed = wide * torch.rsqrt((wide * wide).mean(dim=-1, keepdim=True) + 1e-5) * state["norm"].double()
    g, u = _plain_product(*_quantized(normed), state["weight"]).chunk(2, dim=1)
    return (_act(state["case"]["act"], g) * u).to(torch.bfloat16)


def _capped(scores, cap):
    return cap * torch.tanh(scores / cap) if cap else scores


def _plain_shared(state):
    case = state["case"]
    heads, kv, dim, scale, cap = case["heads"], case["kv_heads"], case["dim"], state["scale"], case["softcap"]
    per, live = heads // kv, state["positions"].numel() - case["idle"]
    q = state["q"][:live].float().view(live, kv, per, dim)
    positions, segment = state["positions"][:live].long(), state["segment"][:live].long()
    starts, pages, table = state["starts"].long(), state["pages"].long(), state["table"].long()
    group = torch.searchsorted(starts, torch.arange(live, device=DEVICE), right=True) - 1
    # the shared keys, once a group: its tokens as rows of one product
    row = starts[:-1, None] + torch.arange(state["most_tokens"], device=DEVICE)[None, :]
    here = row < starts[1:, None]
    row = row.clamp(max=live - 1)
    front = table[segment[starts[:-1]], :state["most_pages"]].clamp(min=0)
    k = state["k"][front].float().permute(0, 2, 1, 3, 4).flatten(2, 3)           # [group][kv][key][dim]
    v = state["v"][front].float().permute(0, 2, 1, 3, 4).flatten(2, 3)
    key = torch.arange(state["most_pages"] * PAGE, device=DEVICE)
    seen = (key[None, None, :] < PAGE * pages[:, None, None]) & (key[None, None, :] <= positions[row][:, :, None])
    wide = q[row].permute(0, 2, 1, 3, 4).flatten(2, 3)                           # [group][kv][token x per][dim]
    scores = _capped((wide @ k.transpose(2, 3)) * scale, cap)
    scores = scores.masked_fill(~seen.repeat_interleave(per, dim=1)[:, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    weight = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    back = torch.zeros(live, dtype=torch.long, device=DEVICE)
    back[row[here]] = torch.nonzero(here.flatten()).flatten()                    # a token's place among the groups' rows

    def of_tokens(t):
        return t.view(t.shape[0], kv, -1, per, t.shape[-1]).permute(0, 2, 1, 3, 4).flatten(0, 1)[back]

    o, top, total = of_tokens(weight @ v), of_tokens(top), of_tokens(weight.sum(dim=-1, keepdim=True))
    # every request's own keys
    key = PAGE * pages[group][:, None] + torch.arange(state["most_own"], device=DEVICE)[None, :]
    page = table[segment[:, None], (key // PAGE).clamp(max=table.shape[1] - 1)].clamp(min=0)
    k, v = state["k"][page, :, key % PAGE].float(), state["v"][page, :, key % PAGE].float()     # [token][key][kv][dim]
    scores = _capped(torch.einsum("tkpd,tnkd->tkpn", q, k) * scale, cap)
    scores = scores.masked_fill((key > positions[:, None])[:, None, None, :], -math.inf)
    both = torch.maximum(top, scores.amax(dim=-1, keepdim=True))
    if state["sink"] is not None:
        both = torch.maximum(both, state["sink"].view(1, kv, per, 1))
    weight, old = torch.exp(scores - both), torch.exp(top - both)
    o = o * old + torch.einsum("tkpn,tnkd->tkpd", weight, v)
    total = total * old + weight.sum(dim=-1, keepdim=True)
    if state["sink"] is not None:
        total = total + torch.exp(state["sink"].view(1, kv, per, 1) - both)
    out = torch.zeros_like(state["q"])
    out[:live] = (o / total).reshape(live, heads * dim).to(out.dtype)
    return out


# ------------------------------------------------------------------ 64 bits
def exact(case, seed):
    global own
    kept, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = kept
    return {"linear": _exact_linear, "gated": _exact_gated, "shared": _exact_shared}[case["kind"]](state)


def _dequantized(x):
    """What the rows' integers stand for."""
    step = (x.abs().max(dim=1, keepdim=True).values / 127).to(torch.float32).to(torch.float64)
    return torch.round(x / step) * step


def _exact_linear(state):
    y = _dequantized(state["x"].to(torch.float64)) @ (state["weight"][0] * state["weight"][1].to(torch.float64)[:, None]).T
    return y + state["residual"].to(torch.float64) if "residual" in state else y


def _exact_gated(state):
    x = state["x"].to(torch.float64)
    x = state["norm"].to(torch.float64) * x / torch.sqrt(torch.mean(x ** 2, dim=1, keepdim=True) + 1e-5)
    y = _dequantized(x) @ (state["weight"][0] * state["weight"][1].to(torch.float64)[:, None]).T
    n = y.shape[1] // 2
    gate, up = y[:, :n], y[:, n:]
    if state["case"]["act"] == "silu":
        return gate / (1 + torch.exp(-gate)) * up
    if state["case"]["act"] == "relu":
        return torch.where(gate > 0, gate, torch.zeros_like(gate)) * up
    return gate * (1 + torch.tanh((2 / math.pi) ** 0.5 * (gate + 0.044715 * gate ** 3))) / 2 * up


def _exact_shared(state):
    """Every token by itself: all of its keys in order, one softmax."""
    case = state["case"]
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    out = torch.zeros(state["q"].shape, dtype=torch.float64, device=DEVICE)
    positions, segment = state["positions"].tolist(), state["segment"].tolist()
    held = None
    for t in range(len(positions) - case["idle"]):
        if segment[t] != held:
            held, span = segment[t], positions[t] + case["tokens"]
            pages = state["table"][held, :-(-span // PAGE)].long().clamp(min=0)
            keys = state["k"][pages].transpose(1, 2).flatten(0, 1).transpose(0, 1).to(torch.float64)     # [kv][key][dim]
            values = state["v"][pages].transpose(1, 2).flatten(0, 1).transpose(0, 1).to(torch.float64)
        n = positions[t] + 1
        q = state["q"][t].to(torch.float64).view(kv, heads // kv, dim)
        scores = torch.bmm(q, keys[:, :n].transpose(1, 2)) * state["scale"]
        if case["softcap"]:
            scores = torch.tanh(scores / case["softcap"]) * case["softcap"]
        if state["sink"] is not None:
            scores = torch.cat([scores, state["sink"].to(torch.float64).view(kv, heads // kv, 1)], dim=2)
        p = torch.softmax(scores, dim=2)
        out[t] = torch.bmm(p[:, :, :n], values[:, :n]).flatten()
    return out
