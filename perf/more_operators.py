"""The routed experts of a mixture-of-experts MLP in W8A8, as measurable cases: what a serving program does between the
router's logits and the layer's output.

* ``route``: each token's experts and their weights from the router's logits, and the order in which the experts work
  through the tokens.
* ``linear``: one Linear per expert on the rows of that expert, any number of rows each, as one grouped product of codes.
* ``swiglu``: the experts' up and gate projections with the activation between them.
* ``combine``: the experts' outputs back in the tokens' order, weighted and summed.
* ``moe``: all of it, as a layer's forward calls it.

Activations are bf16 or fp32, weights int8 codes ``[experts, out, in]`` with a scale per output channel.  The package is inference only: there is no
backward direction.
"""
import math

import torch

own = False
DEVICE = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _route(name, tokens, experts, k, dtype="bf16", masked=False, renormalize=True):
    return dict(name=name, kind="route", tokens=tokens, experts=experts, k=k, dtype=dtype, masked=masked, renormalize=renormalize)


def _linear(name, tokens, experts, k, dim, out, dtype="bf16", gather=True, bias=False):
    return dict(name=name, kind="linear", tokens=tokens, experts=experts, k=k, dim=dim, out=out, dtype=dtype, gather=gather, bias=bias)


def _swiglu(name, tokens, experts, k, dim, ffn, dtype="bf16"):
    return dict(name=name, kind="swiglu", tokens=tokens, experts=experts, k=k, dim=dim, ffn=ffn, dtype=dtype)


def _combine(name, tokens, experts, k, dim, dtype="bf16", masked=False, residual=False):
    return dict(name=name, kind="combine", tokens=tokens, experts=experts, k=k, dim=dim, dtype=dtype, masked=masked, residual=residual)


def _moe(name, tokens, experts, k, dim, ffn, masked=False, residual=False):
    return dict(name=name, kind="moe", tokens=tokens, experts=experts, k=k, dim=dim, ffn=ffn, masked=masked, residual=residual)


def listed():
    return [
        # a padded batch of short prompts, float logits
        _route("route_333x4_of_60_f32_masked", 333, 60, 4, "f32", masked=True),
        # a long prompt over many small experts; weights as the softmax over all of them gives them
        _route("route_16384x8_of_256", 16384, 256, 8, renormalize=False),
        # a small decode batch in fp32, an odd number of outputs
        _linear("linear_5x2_of_8_f32_bias", 5, 8, 2, 1536, 1001, "f32", bias=True),
        # the experts' second projection of a large prefill: rows already in the experts' order
        _linear("linear_8000x6_of_64_rows", 8000, 64, 6, 1408, 2048, gather=False),
        # a decode batch: most experts have one row or two
        _swiglu("swiglu_24x4_of_60", 24, 60, 4, 2048, 1408),
        # a prompt of the 1536-wide model
        _swiglu("swiglu_2000x6_of_64", 2000, 64, 6, 1536, 1408),
        # a decode batch
        _combine("combine_11x6", 11, 64, 6, 2048),
        # a large padded prefill beside shared experts, whose output is the residual
        _combine("combine_16384x8_masked_residual", 16384, 64, 8, 2048, masked=True, residual=True),
        # one sequence, one token
        _moe("moe_1x6_of_64", 1, 64, 6, 2048, 1408),
        # a decode batch
        _moe("moe_16x6_of_64", 16, 64, 6, 2048, 1408),
        # a padded batch of prompts through few large experts of the 1536-wide model's MLP
        _moe("moe_500x2_of_8_masked_residual", 500, 8, 2, 1536, 6912, masked=True, residual=True),
        # a prompt
        _moe("moe_4096x6_of_64", 4096, 64, 6, 2048, 1408),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _experts(rng):
    experts = rng.choice((2, 4, 8, 16, 32, 60, 64, 100, 128, 160, 256))
    return experts, rng.randint(1, min(8, experts))


def _most_tokens(rng, most, each):
    """Up to `most` tokens, of which each costs `each` of the largest case's 4.3e11 operations."""
    return _log(rng, 1, max(1, min(most, int(4.0e11 / each))))


def _draw_route(rng):
    experts, k = _experts(rng)
    return _route("", _log(rng, 1, 16384), experts, k, rng.choice(("bf16", "f32")), rng.random() < 0.4, rng.random() < 0.6)


def _draw_linear(rng):
    experts, k = _experts(rng)
    dim, out = 16 * _log(rng, 8, 256), _log(rng, 40, 4096)
    while experts * dim * out > 6e8:
        experts = max(experts // 2, k)
        out = max(40, out * 3 // 4)
    return _linear("", _most_tokens(rng, 8000, 2 * k * dim * out), experts, k, dim, out, rng.choice(("bf16", "bf16", "f32")), rng.random() < 0.5, rng.random() < 0.3)


def _draw_swiglu(rng):
    experts, k = _experts(rng)
    dim, ffn = 16 * _log(rng, 8, 256), 16 * _log(rng, 4, 256)
    while experts * dim * ffn * 2 > 6e8:
        experts = max(experts // 2, k)
        ffn = 16 * max(4, ffn * 3 // 64)
    return _swiglu("", _most_tokens(rng, 8000, 4 * k * dim * ffn), experts, k, dim, ffn, rng.choice(("bf16", "bf16", "f32")))


def _draw_combine(rng):
    experts, k = _experts(rng)
    dim = 16 * _log(rng, 8, 256)
    return _combine("", _log(rng, 1, min(16384, int(2.6e8 / (k * dim)))), experts, k, dim, rng.choice(("bf16", "bf16", "f32")), rng.random() < 0.4, rng.random() < 0.5)


def _draw_moe(rng):
    experts, k = _experts(rng)
    dim, ffn = 16 * _log(rng, 16, 256), 16 * _log(rng, 8, 432)
    while experts * dim * ffn * 3 > 6e8:
        experts = max(experts // 2, k)
        ffn = 16 * max(8, ffn * 3 // 64)
    return _moe("", _most_tokens(rng, 6000, 6 * k * dim * ffn), experts, k, dim, ffn, rng.random() < 0.4, rng.random() < 0.4)


def draw(rng):
    case = rng.choices((_draw_route, _draw_linear, _draw_swiglu, _draw_combine, _draw_moe), (2, 3, 2, 2, 5))[0](rng)
    del case["name"]
    return case


# ---- what is in hand before the call -----------------------------------------------------------------------------

def _logits(case, gen, dtype):
    """As a trained router gives them: some experts are asked more often than others; a padded token has no expert."""
    tokens, experts = case["tokens"], case["experts"]
    x = torch.randn(tokens, experts, generator=gen, device=DEVICE) * 1.5 + torch.randn(experts, generator=gen, device=DEVICE) * 0.5
    if case.get("masked"):
        x[torch.rand(tokens, generator=gen, device=DEVICE) < 0.2] = -math.inf
    return x.to(dtype)


def _codes(gen, *shape):
    return torch.empty(*shape, device=DEVICE, dtype=torch.bfloat16).normal_(std=36.0, generator=gen).round_().clamp_(-127, 127).to(torch.int8)


def _scales(gen, size, *shape):
    return torch.empty(*shape, device=DEVICE).normal_(std=0.25, generator=gen).exp_().mul_(size)


def _weight(gen, experts, out, dim):
    return _codes(gen, experts, out, dim), _scales(gen, 1 / (36.0 * math.sqrt(dim)), experts, out)


def _grouped(case, gen):
    """Tokens dealt out to experts: the experts' offsets and the token of each row, as the router leaves them."""
    s = _plain_route({"logits": _logits(case, gen, torch.float32), "k": case["k"], "renormalize": True})
    return {"offsets": s["offsets"], "tokens": s["tokens"]}, s


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, dtype = case["kind"], TYPES[case.get("dtype", "bf16")]
    s = {"kind": kind, "k": case["k"]}
    if kind == "route":
        return {**s, "logits": _logits(case, gen, dtype), "renormalize": case["renormalize"]}
    if kind == "combine":
        rows = case["tokens"] * case["k"]
        y = torch.empty(rows, case["dim"], device=DEVICE, dtype=dtype).normal_(generator=gen)
        r = _grouped(case, gen)[1]
        res = torch.empty(case["tokens"], case["dim"], device=DEVICE, dtype=dtype).normal_(generator=gen) if case["residual"] else None
        return {**s, "y": y, "rows": r["rows"], "weights": r["weights"], "residual": res}
    if kind in ("linear", "swiglu"):
        out = case["out"] if kind == "linear" else 2 * case["ffn"]
        groups, _ = _grouped(case, gen)
        rows = case["tokens"]
        if kind == "linear" and not case["gather"]:
            rows, groups["tokens"] = rows * case["k"], None
        wq, sw = _weight(gen, case["experts"], out, case["dim"])
        bias = torch.randn(case["experts"], out, generator=gen, device=DEVICE).to(dtype) if case.get("bias") else None
        return {**s, **groups, "xq": _codes(gen, rows, case["dim"]), "sx": _scales(gen, 1 / 36.0, rows), "wq": wq, "sw": sw, "bias": bias, "dtype": dtype}
    x = torch.randn(case["tokens"], case["dim"], generator=gen, device=DEVICE)
    x[:, 5] *= 6.0  # as trained models have it: a loud channel
    up_gate, down = _weight(gen, case["experts"], 2 * case["ffn"], case["dim"]), _weight(gen, case["experts"], case["dim"], case["ffn"])
    res = torch.randn(case["tokens"], case["dim"], generator=gen, device=DEVICE).to(dtype) if case["residual"] else None
    return {**s, "x": x.to(dtype), "logits": _logits(case, gen, dtype), "up_gate": up_gate, "down": down, "residual": res, "dtype": dtype}


# ---- the call ------------------------------------------------------------------------------------------------------

def _plain_route(s):
    x, k = s["logits"].float(), s["k"]
    tokens, experts = x.shape
    top, at = torch.sort(x, dim=1, descending=True, stable=True)  # equal logits: the lowest expert first
    top, at = top[:, :k], at[:, :k]
    there = top > -math.inf
    most = torch.where(there[:, :1], top[:, :1], 0.0)
    e = torch.exp(torch.where(there, top, -math.inf) - most)
    total = (e if s["renormalize"] else torch.exp(x - most)).sum(1, keepdim=True)
    weights = torch.where(there, e / total, 0.0)
    group = torch.where(there, at, experts).reshape(-1)
    grouped, order = torch.sort(group, stable=True)
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=x.device)
    offsets = torch.searchsorted(grouped, torch.arange(experts + 1, device=x.device))
    return {"weights": weights, "experts": torch.where(there, at, -1).int(), "rows": torch.where(there, place.view(tokens, k), -1).int(),
            "tokens": torch.where(grouped < experts, order // k, -1).int(), "offsets": offsets.int()}


def _plain_grouped(xq, sx, wq, sw, offsets, tokens, bias, dtype):
    """Row by row with its expert's weight where rows are few, expert by expert otherwise.  Sums of these codes stay below 2^24: exact in fp32."""
    out = wq.shape[1]
    rows = xq.shape[0] if tokens is None else tokens.numel()
    group = torch.searchsorted(offsets, torch.arange(rows, device=xq.device, dtype=torch.int32), right=True) - 1
    if tokens is not None:
        xq, sx = xq[tokens], sx[tokens]
    if rows * out * xq.shape[1] <= 1 << 27:
        acc = torch.matmul(wq[group].float(), xq.float().unsqueeze(2)).squeeze(2)
    else:
        acc = torch.empty(rows, out, device=xq.device)
        at = offsets.tolist()
        for e in range(len(at) - 1):
            if at[e + 1] > at[e]:
                acc[at[e]:at[e + 1]] = xq[at[e]:at[e + 1]].float() @ wq[e].float().t()
    y = (acc * sx[:, None]) * sw[group]
    return (y if bias is None else y + bias[group].float()).to(dtype)


def _plain_swiglu(ug):
    up, gate = ug.float().chunk(2, dim=1)
    return (up * (gate / (1.0 + torch.exp(-gate)))).to(ug.dtype)


def _plain_combine(y, rows, weights, residual):
    live = rows >= 0
    out = (torch.where(live[:, :, None], y[rows.clamp(min=0)].float(), 0.0) * weights[:, :, None]).sum(1)
    return (out if residual is None else out + residual.float()).to(y.dtype)


def _plain_quantise(x):
    x = x.float()
    most = x.abs().amax(1)
    scale = torch.where(most > 0, most / 127.0, 1.0)
    return torch.round(x / scale[:, None]).clamp(-127, 127).to(torch.int8), scale


def _plain_moe(s):
    r = _plain_route({**s, "renormalize": True})
    xq, sx = _plain_quantise(s["x"])
    live = r["tokens"][:int(r["offsets"][-1])]
    h = _plain_swiglu(_plain_grouped(xq, sx, *s["up_gate"], r["offsets"], live, None, s["dtype"]))
    hq, sh = _plain_quantise(h)
    y = _plain_grouped(hq, sh, *s["down"], r["offsets"], None, None, s["dtype"])
    if not live.numel():
        return torch.zeros_like(s["x"]) if s["residual"] is None else s["residual"].clone()
    return _plain_combine(y, r["rows"], r["weights"], s["residual"])


def run(state):
    s, kind = state, state["kind"]
    if own:
        from khaosz_amd import ops

        if kind == "route":
            return ops.route_topk(s["logits"], s["k"], renormalize=s["renormalize"])._asdict()
        if kind == "linear":
            return ops.linear_w8a8_grouped(s["xq"], s["sx"], s["wq"], s["sw"], s["offsets"], s["tokens"], bias=s["bias"], out_dtype=s["dtype"])
        if kind == "swiglu":
            return ops.swiglu_w8a8_grouped(s["xq"], s["sx"], s["wq"], s["sw"], s["offsets"], s["tokens"], out_dtype=s["dtype"])
        if kind == "combine":
            return ops.combine_rows(s["y"], s["rows"], s["weights"], residual=s["residual"])
        return ops.experts_w8a8(s["x"], ops.route_topk(s["logits"], s["k"]), *s["up_gate"], *s["down"], residual=s["residual"])
    if kind == "route":
        return _plain_route(s)
    if kind == "combine":
        return _plain_combine(s["y"], s["rows"], s["weights"], s["residual"])
    if kind == "moe":
        return _plain_moe(s)
    y = _plain_grouped(s["xq"], s["sx"], s["wq"], s["sw"], s["offsets"], s["tokens"], s["bias"], s["dtype"])
    return y if kind == "linear" else _plain_swiglu(y)


# ---- what it cannot do without -----------------------------------------------------------------------------------

def work(case):
    tokens, experts, k = case["tokens"], case["experts"], case["k"]
    size = 4 if case.get("dtype") == "f32" else 2
    rows = tokens * k * (0.8 if case.get("masked") else 1.0)
    used = experts * (1 - (1 - k / experts) ** (rows / k))  # experts with a row, as if all were asked alike
    kind = case["kind"]
    if kind == "route":
        return {"bytes": tokens * experts * size + 16 * tokens * k + 4 * (experts + 1), "flops": 0}
    if kind == "combine":
        return {"bytes": (rows + tokens * (2 if case["residual"] else 1)) * case["dim"] * size + 8 * tokens * k, "flops": 2.0 * rows * case["dim"]}
    dim = case["dim"]
    if kind == "moe":
        ffn = case["ffn"]
        return {"bytes": used * 3 * dim * ffn + tokens * dim * size * (3 if case["residual"] else 2) + tokens * experts * size, "flops": 6.0 * rows * dim * ffn}
    out = case["out"] if kind == "linear" else 2 * case["ffn"]
    written = rows * (out if kind == "linear" else out // 2) * size
    read = (tokens if kind == "swiglu" or case["gather"] else rows) * dim
    return {"bytes": used * out * dim + read + written, "flops": 2.0 * rows * dim * out}


# ---- the definitions, in 64 bits -----------------------------------------------------------------------------------

def _exact_route(logits, k, renormalize):
    tokens, experts = logits.shape
    x = logits.double()
    chosen = torch.full((tokens, experts), -1, device=DEVICE)
    for t in range(0, tokens, 1024):  # an expert's place in its token's order: how many are larger, or equal and before it
        a, b = x[t:t + 1024, :, None], x[t:t + 1024, None, :]
        before = torch.ones(experts, experts, device=DEVICE, dtype=torch.bool).tril(-1)
        chosen[t:t + 1024] = ((b > a) | ((b == a) & before)).sum(2)
    picked = (chosen < k) & torch.isfinite(x)
    experts_of = torch.full((tokens, k), -1, device=DEVICE)
    t, e = picked.nonzero(as_tuple=True)
    j = chosen[t, e]
    experts_of[t, j] = e
    counts = picked.sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = offsets[:-1] + picked.cumsum(0) - 1
    rows = torch.full_like(experts_of, -1)
    rows[t, j] = place[t, e]
    tokens_of = torch.full((tokens * k,), -1, device=DEVICE)
    tokens_of[place[t, e]] = t
    p = torch.softmax(x, 1).nan_to_num(0.0)
    weights = torch.zeros(tokens, k, device=DEVICE, dtype=torch.float64)
    weights[t, j] = p[t, e]
    if renormalize:
        weights = (weights / weights.sum(1, keepdim=True)).nan_to_num(0.0)
    return {"weights": weights, "experts": experts_of.int(), "rows": rows.int(), "tokens": tokens_of.int(), "offsets": offsets.int()}


def _exact_rows(codes, scale, wq, sw, expert_rows, out_rows, bias=None):
    """expert_rows: for each expert the rows of `codes` it works on."""
    y = torch.zeros(out_rows, wq.shape[1], device=DEVICE, dtype=torch.float64)
    at = 0
    for e, rows in enumerate(expert_rows):
        if len(rows):
            p = torch.matmul(codes[rows].double() * scale[rows].double()[:, None], wq[e].double().t().contiguous()) * sw[e].double()
            y[at:at + len(rows)] = p if bias is None else p + bias[e].double()
            at += len(rows)
    return y


def _exact_swiglu(ug, dtype):
    up, gate = ug.to(dtype).double().chunk(2, dim=1)  # up and gate are values of the output's type
    return up * torch.sigmoid(gate) * gate


def _exact_codes(x):
    """The definition's codes: the scale and the quotient are 32-bit numbers (a double's quotient of two, rounded, is theirs)."""
    x = x.double()
    most = x.abs().max(dim=1).values
    scale = torch.where(most > 0, (most / 127.0).float(), torch.ones_like(most, dtype=torch.float32))
    return torch.round((x / scale.double()[:, None]).float().double()), scale


def _exact_moe(s):
    r = _exact_route(s["logits"], s["k"], True)
    tokens, at = r["tokens"].long(), r["offsets"].tolist()
    xq, sx = _exact_codes(s["x"])
    rows = at[-1]
    ug = _exact_rows(xq, sx, *s["up_gate"], [tokens[a:b] for a, b in zip(at, at[1:])], rows)
    hq, sh = _exact_codes(_exact_swiglu(ug, s["dtype"]).to(s["dtype"]))  # h is a value of the activations' type
    y = _exact_rows(hq, sh, *s["down"], [torch.arange(a, b, device=DEVICE) for a, b in zip(at, at[1:])], rows).to(s["dtype"])  # and so is an expert's output
    return _exact_combine(y, r["rows"], r["weights"], s["residual"])


def _exact_combine(y, rows, weights, residual):
    out = torch.zeros(rows.shape[0], y.shape[1], device=DEVICE, dtype=torch.float64) if residual is None else residual.double()
    for j in range(rows.shape[1]):
        t = (rows[:, j] >= 0).nonzero()[:, 0]
        out[t] += y[rows[t, j].long()].double() * weights[t, j].double()[:, None]
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind == "route":
        return _exact_route(s["logits"], s["k"], s["renormalize"])
    if kind == "combine":
        return _exact_combine(s["y"], s["rows"], s["weights"], s["residual"])
    if kind == "moe":
        return _exact_moe(s)
    at = s["offsets"].tolist()
    rows = torch.arange(at[-1], device=DEVICE) if s["tokens"] is None else s["tokens"].long()
    y = _exact_rows(s["xq"], s["sx"], s["wq"], s["sw"], [rows[a:b] for a, b in zip(at, at[1:])], at[-1], s["bias"])
    return y if kind == "linear" else _exact_swiglu(y, s["dtype"])
