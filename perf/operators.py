"""The operators around a packed linear layer, timed: a product with its epilogue, the routing of tokens to experts, and the
experts' products.

A case names one operator, its sizes and its options:

  op "route"      route_experts: the logits of `tokens` tokens over `experts` experts to the `top_k` chosen ones and their weights.
                  `scoring` softmax or sigmoid; `balance`: a bias that takes part in the choice and not in the weights;
                  `groups` / `top_groups`: the choice is among the best groups of experts; the last `padded` tokens have no open expert
  op "product"    StreamingLinear.product: y = act(x w^T + bias) * multiplier + residual of `rows` activation rows, each part if
                  the case has it; w is out_f x in_f, packed
  op "experts"    StreamingExperts: for each of the `top_k` experts e of a token,
                  y += weight * (down_e (act(gate_e x + b) * (up_e x + b)) + b); gate_e and up_e are inner x hidden, stacked in one packed
                  tensor, down_e is hidden x inner.  The last `padded` tokens have no expert

  mix "t"         Student-t weights (nu = 4): nearly all in the first level of (3,5,8)
  mix "real"      integers in the levels of (3,5,8) at 55 / 40 / 5 %, the fractions of trained weights
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
LEVELS = (3, 5, 8)
ACTIVATIONS = ("none", "silu", "gelu", "gelu_tanh", "relu", "relu2")
# The largest of each kind that is listed; drawn cases stay below.
MOST_ROUTED = 16384 * 128
MOST_WEIGHTS = 17408 * 5120
MOST_PRODUCTS = 2048 * MOST_WEIGHTS
MOST_EXPERT_WEIGHTS = 64 * 3 * 2048 * 1024
MOST_EXPERT_PRODUCTS = 4096 * 6 * 3 * 2048 * 1024


def _route(name, tokens, experts, top_k, scoring, dtype, **more):
    case = {"name": name, "op": "route", "tokens": tokens, "experts": experts, "top_k": top_k, "scoring": scoring, "dtype": dtype,
            "balance": False, "groups": 1, "top_groups": 1, "renormalize": True, "scale": 1.0, "padded": 0}
    return {**case, **more}


def _product(name, out_f, in_f, rows, mix, activation, bias, multiplier, residual):
    return {"name": name, "op": "product", "out_f": out_f, "in_f": in_f, "rows": rows, "mix": mix, "activation": activation,
            "bias": bias, "multiplier": multiplier, "residual": residual}


def _experts(name, tokens, experts, top_k, hidden, inner, mix, activation="silu", bias=False, residual=False, padded=0):
    return {"name": name, "op": "experts", "tokens": tokens, "experts": experts, "top_k": top_k, "hidden": hidden, "inner": inner,
            "mix": mix, "activation": activation, "bias": bias, "residual": residual, "padded": padded}


def listed():
    return [
        # one token of a stream: the smallest call, which a launch's latency bounds
        _route("route_token", 1, 64, 6, "softmax", "bf16"),
        # a batch of token streams of a balanced router with groups; the batch is padded to its captured size
        _route("route_groups", 96, 160, 6, "sigmoid", "fp32", balance=True, groups=8, top_groups=3, scale=2.5, padded=7),
        # a long prompt, or several together
        _route("route_prompt", 16384, 128, 8, "softmax", "bf16"),
        # a block's last projection of one token, onto the residual stream
        _product("product_token", 5120, 17408, 1, "t", "none", False, False, True),
        # the gate of a gated layer for one token, by the other half's output
        _product("product_gate", 17408, 5120, 1, "real", "silu", False, True, False),
        # several streams, rows that are no whole number of 512-element units, everything at once
        _product("product_batch", 4096, 11008, 13, "real", "gelu", True, True, True),
        # a prompt of an odd length
        _product("product_prompt", 10240, 5120, 333, "t", "gelu_tanh", True, False, True),
        # the gate again, a long prompt
        _product("product_long", 17408, 5120, 2048, "real", "silu", False, True, False),
        # a token through its experts
        _experts("experts_token", 1, 64, 6, 2048, 1024, "real", residual=True),
        # a batch of token streams: nearly every expert has some, and none has many
        _experts("experts_batch", 64, 64, 6, 2048, 1024, "t", residual=True),
        # few experts of sizes that are no whole tiles, biases, and a padded prompt
        _experts("experts_odd", 205, 20, 3, 1400, 744, "real", activation="gelu_tanh", bias=True, padded=5),
        # a long prompt: every expert has some hundred tokens
        _experts("experts_prompt", 4096, 64, 6, 2048, 1024, "real", residual=True),
    ]


def _log(rng, lo, hi):
    return math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))


def _size(rng, lo, hi, steps):
    v, step = _log(rng, lo, hi), rng.choice(steps)
    return max(step, min(int(round(v / step)) * step, hi // step * step))


def draw(rng):
    """Tokens and rows from one on, sizes in whole tiles, in whole pieces of 8 and now and then of any length."""
    op = rng.choice(("route", "product", "experts"))
    if op == "route":
        groups = rng.choice((1, 1, 1, 2, 4, 8))
        experts = groups * int(round(_log(rng, max(8 / groups, 2), 512 / groups)))
        top_groups = rng.randint((groups + 1) // 2, groups)
        tokens = int(round(_log(rng, 1, min(16384, MOST_ROUTED // experts))))
        scoring = rng.choice(("softmax", "sigmoid"))
        return _route("", tokens, experts, rng.randint(1, min(16, top_groups * (experts // groups))), scoring, rng.choice(("bf16", "fp16", "fp32")),
                      balance=rng.random() < 0.5, groups=groups, top_groups=top_groups, renormalize=rng.random() < 0.7,
                      scale=rng.choice((1.0, 2.5)), padded=rng.choice((0, 0, tokens // 9))) | {"name": None}
    if op == "product":
        in_f = _size(rng, 256, 17408, (512, 512, 8, 8, 1))
        out_f = _size(rng, 128, min(17408, max(128, MOST_WEIGHTS // in_f)), (32, 32, 8, 1))
        rows = 1
        if rng.random() < 0.7:
            rows = int(round(_log(rng, 2, min(2048, MOST_PRODUCTS // (out_f * in_f)))))
        return _product(None, out_f, in_f, rows, rng.choice(("t", "real")), rng.choice(ACTIVATIONS), rng.random() < 0.4,
                        rng.random() < 0.4, rng.random() < 0.5)
    hidden = _size(rng, 256, 4096, (512, 64, 64, 8, 1))
    inner = _size(rng, 96, 2048, (64, 64, 8, 1))
    experts = int(round(_log(rng, 4, max(4, min(128, MOST_EXPERT_WEIGHTS // (3 * hidden * inner))))))
    top_k = rng.randint(1, min(8, experts))
    tokens = int(round(_log(rng, 1, min(4096, MOST_EXPERT_PRODUCTS // (3 * hidden * inner * top_k)))))
    return _experts(None, tokens, experts, top_k, hidden, inner, rng.choice(("t", "real")), rng.choice(ACTIVATIONS[1:4]),
                    rng.random() < 0.3, rng.random() < 0.5, rng.choice((0, 0, tokens // 9)))


# ---------------------------------------------------------------------------------------------------------------------
#  inputs
# ---------------------------------------------------------------------------------------------------------------------
def _t_tail(t):
    """P(|T| > t) for four degrees of freedom."""
    q = t * t / (1 + t * t / 4)
    return 1 - 0.75 * math.sqrt(q) * (1 - q / 12)


def _t_largest(n):
    """The median of the largest |T| of n."""
    lo, hi = 1.0, 1e4
    for _ in range(60):
        mid = math.sqrt(lo * hi)
        lo, hi = (mid, hi) if n * _t_tail(mid) > math.log(2) else (lo, mid)
    return lo


def _weights(n_matrices, out_f, in_f, mix, gen):
    """bf16 weights before they are packed, [n_matrices, out_f, in_f]; their size is about that of one over the root of in_f."""
    n = out_f * in_f
    out = torch.empty((n_matrices, n), dtype=torch.bfloat16, device=DEV)
    for w_out in out:
        at = int(torch.randint(n, (1,), generator=gen, device=DEV))
        if mix == "t":
            z = torch.randn(n, generator=gen, device=DEV)
            chi = torch.randn(n, generator=gen, device=DEV).square_()
            for _ in range(3):
                chi += torch.randn(n, generator=gen, device=DEV).square_()
            w = z.div_(chi.div_(4).sqrt_())
            top = _t_largest(n)  # the largest weight sets the scale and so the level shares
            w.clamp_(-top, top)
            w[at] = top
            w.mul_((0.5 / in_f) ** 0.5)
        else:  # levels drawn, magnitudes uniform within a level; one 127 fixes the scale
            u = torch.rand(n, generator=gen, device=DEV)
            f = torch.rand(n, generator=gen, device=DEV)
            w = torch.where(u < 0.55, (f * 4).floor_(), torch.where(u < 0.95, (f * 12).floor_() + 4, (f * 112).floor_() + 16))
            w.mul_((torch.rand(n, generator=gen, device=DEV) < 0.5).mul(2).sub(1))
            w[at] = 127
            w.mul_(float(torch.tensor(in_f ** -0.5 / 18).bfloat16()))
        w_out.copy_(w)
    return out.view(n_matrices, out_f, in_f)


def _decoded(weights):
    """What packing makes of bf16 weights, a matrix at a time: integers of 8 bits by a bf16 scale, as bf16."""
    out = torch.empty_like(weights)
    for w, o in zip(weights, out):
        scale = w.abs().max().clamp(min=1e-8) / 127.0
        o.copy_((w.float() / scale).round().clamp(-127, 127) * scale.float())
    return out


def _normal(shape, gen, by=1.0, dtype=torch.bfloat16):
    return torch.randn(shape, generator=gen, device=DEV).mul_(by).to(dtype)


def _assignments(case, gen):
    """The experts of each token and their weights as a router gives them: some experts are liked more than others."""
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    logits = torch.randn((tokens, experts), generator=gen, device=DEV) + 0.5 * torch.randn(experts, generator=gen, device=DEV)
    top, ids = logits.topk(top_k, dim=1)
    weights = torch.exp(top - top[:, :1])
    weights = weights / weights.sum(1, keepdim=True)
    ids = ids.to(torch.int32)
    if case["padded"]:
        ids[tokens - case["padded"]:] = -1
        weights[tokens - case["padded"]:] = 0
    return ids, weights


def _inputs(case, seed):
    """Everything a case is computed from; weights before they are packed."""
    gen = torch.Generator(DEV).manual_seed(seed)
    op = case["op"]
    if op == "route":
        dtype = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[case["dtype"]]
        logits = _normal((case["tokens"], case["experts"]), gen, 1.5, dtype)
        if case["padded"]:
            logits[case["tokens"] - case["padded"]:] = -math.inf
        bias = _normal(case["experts"], gen, 0.1, torch.float32) if case["balance"] else None
        return {"logits": logits, "bias": bias}
    if op == "product":
        rows, in_f, out_f = case["rows"], case["in_f"], case["out_f"]
        return {"w": _weights(1, out_f, in_f, case["mix"], gen), "x": _normal((rows, in_f), gen),
                "bias": _normal(out_f, gen, 0.3) if case["bias"] else None,
                "multiplier": _normal((rows, out_f), gen) if case["multiplier"] else None,
                "residual": _normal((rows, out_f), gen) if case["residual"] else None}
    tokens, experts, hidden, inner = case["tokens"], case["experts"], case["hidden"], case["inner"]
    ids, weights = _assignments(case, gen)
    return {"gate_up": _weights(experts, 2 * inner, hidden, case["mix"], gen), "down": _weights(experts, hidden, inner, case["mix"], gen),
            "gate_up_bias": _normal((experts, 2 * inner), gen, 0.3) if case["bias"] else None,
            "down_bias": _normal((experts, hidden), gen, 0.3) if case["bias"] else None,
            "x": _normal((tokens, hidden), gen), "ids": ids, "weights": weights,
            "residual": _normal((tokens, hidden), gen) if case["residual"] else None}


@torch.no_grad()
def prepare(case, seed):
    state = {"case": dict(case), **_inputs(case, seed)}
    op = case["op"]
    if op == "product":
        if own:
            from ixrun_amd import Int8XEngine

            layer = torch.nn.Linear(case["in_f"], case["out_f"], bias=case["bias"], device="meta", dtype=torch.bfloat16)
            layer.weight = torch.nn.Parameter(state.pop("w")[0], requires_grad=False)
            if case["bias"]:
                layer.bias = torch.nn.Parameter(state["bias"], requires_grad=False)
            model = torch.nn.ModuleList([layer])
            Int8XEngine._deploy_streaming(model, LEVELS, verbose=False)
            state["layer"] = model[0]
        else:
            state["w"] = _decoded(state["w"])[0]
    if op == "experts":
        gate_up, down = state.pop("gate_up"), state.pop("down")
        if own:
            from ixrun_amd import StreamingExperts

            state["layer"] = StreamingExperts.from_weights(gate_up, down, level_bits=LEVELS, activation=case["activation"],
                                                           gate_up_bias=state["gate_up_bias"], down_bias=state["down_bias"])
        else:
            state.update(gate_up=_decoded(gate_up), down=_decoded(down))
    return state


# ---------------------------------------------------------------------------------------------------------------------
#  one pass
# ---------------------------------------------------------------------------------------------------------------------
def _activated(v, name):
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5))
    if name == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh((2 / math.pi) ** 0.5 * (v + 0.044715 * v * v * v)))
    if name == "relu":
        return v.clamp(min=0)
    if name == "relu2":
        return v.clamp(min=0).square()
    return v


def _plain_route(state):
    case = state["case"]
    logits, top_k, groups = state["logits"].double(), case["top_k"], case["groups"]
    tokens, experts = logits.shape
    is_open = logits != -math.inf
    if case["scoring"] == "softmax":
        most = logits.amax(1, keepdim=True)
        scores = torch.where(is_open, torch.exp(logits - torch.where(most == -math.inf, 0.0, most)), 0.0)
        scores = scores / scores.sum(1, keepdim=True).clamp(min=torch.finfo(torch.float64).tiny)
    else:
        scores = torch.where(is_open, 1 / (1 + torch.exp(-logits)), 0.0)
    # without a bias the choice is by the logits, whose order is that of the scores
    choice = logits if state["bias"] is None else torch.where(is_open, scores + state["bias"].double(), -math.inf)
    if groups > 1:
        by_group = choice.view(tokens, groups, experts // groups)
        if state["bias"] is None:
            group_score = by_group.amax(2)
        else:
            best = torch.sort(by_group, dim=2, descending=True)[0][:, :, :2]
            group_score = torch.where(best[:, :, 0] == -math.inf, best[:, :, 0], torch.where(best == -math.inf, 0.0, best).sum(2))
        kept = torch.sort(group_score, dim=1, descending=True, stable=True)[1][:, :case["top_groups"]]
        mask = torch.zeros((tokens, groups), dtype=torch.bool, device=logits.device).scatter_(1, kept, True)
        choice = torch.where(mask.repeat_interleave(experts // groups, dim=1), choice, -math.inf)
    top, ids = torch.sort(choice, dim=1, descending=True, stable=True)
    top, ids = top[:, :top_k], ids[:, :top_k]
    taken = top != -math.inf
    weights = torch.where(taken, scores.gather(1, ids), 0.0)
    if case["renormalize"]:
        weights = weights / weights.sum(1, keepdim=True).clamp(min=torch.finfo(torch.float64).tiny)
    return torch.where(taken, ids, -1).to(torch.int32), (weights * case["scale"]).float()


def _plain_product(state):
    y = state["x"].float() @ state["w"].float().t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    y = _activated(y, state["case"]["activation"])
    if state["multiplier"] is not None:
        y = y * state["multiplier"].float()
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(torch.bfloat16)


def _plain_experts(state):
    case = state["case"]
    x, top_k, inner = state["x"], case["top_k"], case["inner"]
    flat = state["ids"].reshape(-1).long()
    order = torch.sort(flat, stable=True)[1]
    counts = torch.bincount(flat + 1, minlength=case["experts"] + 1).tolist()
    per_slot = torch.zeros((flat.numel(), case["hidden"]), dtype=torch.float32, device=x.device)
    at = counts[0]  # the slots without an expert
    for e, n in enumerate(counts[1:]):
        if n == 0:
            continue
        slots = order[at:at + n]
        at += n
        v = x[slots // top_k].float() @ state["gate_up"][e].float().t()
        if state["gate_up_bias"] is not None:
            v = v + state["gate_up_bias"][e].float()
        v = _activated(v[:, :inner], case["activation"]) * v[:, inner:]
        v = v @ state["down"][e].float().t()
        if state["down_bias"] is not None:
            v = v + state["down_bias"][e].float()
        per_slot[slots] = v
    y = (per_slot.view(-1, top_k, case["hidden"]) * state["weights"].unsqueeze(2)).sum(1)
    if state["residual"] is not None:
        y = y + state["residual"].float()
    return y.to(torch.bfloat16)


@torch.no_grad()
def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        return {"route": _plain_route, "product": _plain_product, "experts": _plain_experts}[op](state)
    if op == "route":
        from ixrun_amd import route_experts

        return route_experts(state["logits"], case["top_k"], scoring=case["scoring"], bias=state["bias"], n_groups=case["groups"],
                             top_groups=case["top_groups"], renormalize=case["renormalize"], scale=case["scale"])
    if op == "product":
        return state["layer"].product(state["x"], activation=case["activation"], multiplier=state["multiplier"], residual=state["residual"])
    return state["layer"](state["x"], state["ids"], state["weights"], residual=state["residual"])


# ---------------------------------------------------------------------------------------------------------------------
#  the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_activation(v, name):
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return v * torch.special.ndtr(v)
    if name == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    if name in ("relu", "relu2"):
        return torch.relu(v) ** (2 if name == "relu2" else 1)
    return v


@torch.no_grad()
def exact(case, seed):
    inp = _inputs(case, seed)
    op = case["op"]
    if op == "route":  # the weights of the chosen experts; which are chosen has no value in between
        l = inp["logits"].double()
        p = torch.softmax(l, 1) if case["scoring"] == "softmax" else torch.sigmoid(l)
        p = torch.nan_to_num(p)  # (tokens without an open expert)
        choice = torch.where(l == -math.inf, l, (p if inp["bias"] is not None else l) + (0 if inp["bias"] is None else inp["bias"].double()))
        if case["groups"] > 1:
            parts = choice.view(*l.shape[:1], case["groups"], -1)
            n = 1 if inp["bias"] is None else min(2, parts.shape[2])
            score = parts.topk(n, 2)[0].sum(2)
            place = torch.argsort(torch.argsort(score, dim=1, descending=True, stable=True), dim=1)
            choice = torch.where((place < case["top_groups"]).unsqueeze(2), parts, -math.inf).reshape(l.shape)
        top, ids = choice.topk(case["top_k"], 1)
        w = p.gather(1, ids) * (top != -math.inf)
        if case["renormalize"]:
            w = torch.nan_to_num(w / w.sum(1, keepdim=True))
        return None, w * case["scale"]
    if op == "product":
        y = inp["x"].double() @ _decoded(inp["w"])[0].double().t()
        y = _exact_activation(y if inp["bias"] is None else y + inp["bias"].double(), case["activation"])
        y = y if inp["multiplier"] is None else y * inp["multiplier"].double()
        return y if inp["residual"] is None else y + inp["residual"].double()
    y = torch.zeros((case["tokens"], case["hidden"]), dtype=torch.float64, device=DEV)
    x = inp["x"].double()
    for e in range(case["experts"]):
        share = torch.where(inp["ids"] == e, inp["weights"].double(), 0.0).sum(1)
        rows = torch.nonzero((inp["ids"] == e).any(1))[:, 0]
        if rows.numel() == 0:
            continue
        both = x[rows] @ _decoded(inp["gate_up"][e:e + 1])[0].double().t()
        if inp["gate_up_bias"] is not None:
            both += inp["gate_up_bias"][e].double()
        gate, up = both.chunk(2, 1)
        v = (_exact_activation(gate, case["activation"]) * up) @ _decoded(inp["down"][e:e + 1])[0].double().t()
        if inp["down_bias"] is not None:
            v += inp["down_bias"][e].double()
        y[rows] += share[rows, None] * v
    return y if inp["residual"] is None else y + inp["residual"].double()


# ---------------------------------------------------------------------------------------------------------------------
#  what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def _beyond(n, mix, edge):
    """Expected share of n weights whose |integer| is above `edge`."""
    if mix == "real":
        return 0.05 * (127 - edge) / 112 if edge >= 15 else 0.05 + 0.4 * (15 - edge) / 12
    return _t_tail((edge + 0.5) * _t_largest(n) / 127)


def _packed_bytes(n, mix):
    bits, left = 0.0, 1.0
    for b in LEVELS[:-1]:
        rest = _beyond(n, mix, (1 << (b - 1)) - 1)
        bits += left + (left - rest) * b
        left = rest
    return n * (bits + 8 * left) / 8 + 2


def work(case):
    op = case["op"]
    if op == "route":
        n, size = case["tokens"] * case["experts"], 4 if case["dtype"] == "fp32" else 2
        return {"bytes": float(n * size + 8 * case["tokens"] * case["top_k"] + (4 * case["experts"] if case["balance"] else 0)),
                "flops": 4.0 * n}
    if op == "product":
        n, rows = case["out_f"] * case["in_f"], case["rows"]
        outs = 1 + case["multiplier"] + case["residual"]
        return {"bytes": _packed_bytes(n, case["mix"]) + 2.0 * rows * (case["in_f"] + outs * case["out_f"]) + 2.0 * case["bias"] * case["out_f"],
                "flops": 2.0 * rows * n}
    hidden, inner, tokens, experts = case["hidden"], case["inner"], case["tokens"] - case["padded"], case["experts"]
    slots = tokens * case["top_k"]
    active = experts * (1 - (1 - case["top_k"] / experts) ** tokens)
    per_expert = _packed_bytes(2 * inner * hidden, case["mix"]) + _packed_bytes(inner * hidden, case["mix"])
    per_expert += 2.0 * case["bias"] * (2 * inner + hidden)
    return {"bytes": active * per_expert + 2.0 * case["tokens"] * hidden * (2 + case["residual"]) + 8.0 * case["tokens"] * case["top_k"],
            "flops": 2.0 * slots * 3 * hidden * inner}
