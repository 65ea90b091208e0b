"""The operators around a packed product from their formulas in 64 bits, with how far a result may be off.

A bound is worked out for each element: u = 2^-24 for a step in fp32, 2^-8 for a rounding to bf16 (half a step, relative), and for a sum of n
terms in fp32, whatever its order, n u times the sum of their magnitudes."""
from __future__ import annotations

import math

import torch

U32, U16 = 2.0 ** -24, 2.0 ** -8
# the largest slope of each activation (relu2's is 2 |v|)
SLOPE = {None: 1.0, "none": 1.0, "silu": 1.1, "gelu": 1.13, "gelu_tanh": 1.13, "relu": 1.0, "relu2": None}


def activation(v, name):
    """In 64 bits."""
    if name == "silu":
        return v * torch.sigmoid(v)
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2))
    if name == "gelu_tanh":
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    if name == "relu":
        return torch.where(v < 0, torch.zeros_like(v), v)
    if name == "relu2":
        return torch.where(v < 0, torch.zeros_like(v), v) ** 2
    return v


def activated(v, off, name):
    """An activation of values that are off by up to `off`, in fp32: its value and how far that is off.

    The formulas take exp, erf or tanh of a value of a few and up to ten steps more: each of these, and the argument's rounding, is a relative
    error of a few u of a factor between 0 and 1 that may be the difference of 1 and something near it, so it is absolute: 16 u |v|."""
    a = activation(v, name)
    slope = SLOPE[name] if SLOPE[name] is not None else 2 * (v.abs() + off)
    return a, slope * off + (0 if name in (None, "none") else 16 * U32 * (v.abs() if name != "relu2" else a))


def product(x, w, bias=None):
    """x w^T + bias in 64 bits, and how far sums in fp32 are off."""
    x, w = x.double(), w.double()
    n = x.shape[-1] + 8
    y, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    return y, n * U32 * size


def rounded(v, off):
    """Values off by up to `off`, rounded to bf16: the rounding of what they should be, and how far another one may be from that.

    Where the interval around a value holds no border between two bf16 the rounding is the same; where it does, it may be a step further."""
    low, high = (v - off).to(torch.bfloat16).double(), (v + off).to(torch.bfloat16).double()
    at = v.to(torch.bfloat16).double()
    return at, torch.maximum(high - at, at - low)


def epilogue(x, w, bias=None, act=None, multiplier=None, residual=None, apart=False):
    """bf16(act(x w^T + bias) * multiplier + residual): value before its rounding, and bound with it.

    `apart`: the product is rounded to bf16 by itself, and its bias added in bf16 (two roundings of what is at most the sum of both)."""
    y, off = product(x, w, bias)
    if apart:
        off = off + 2 * U16 * (1 + U16) * (y.abs() + off + (bias.double().abs() if bias is not None else 0))
    y, off = activated(y, off, act)
    if multiplier is not None:
        m = multiplier.double()
        y, off = y * m, off * m.abs() + U32 * (y * m).abs()
    if residual is not None:
        y = y + residual.double()
        off = off + U32 * y.abs()
    return y, off + U16 * (y.abs() + off)


def experts(x, ids, weights, gate_up, down, act="silu", gated=True, gate_up_bias=None, down_bias=None, residual=None):
    """StreamingExperts over dequantised weights [n, rows, hidden] and [n, hidden, inner]."""
    n, hidden = down.shape[0], down.shape[1]
    x2, ids, weights = x.reshape(-1, hidden), ids.reshape(-1, ids.shape[-1]), weights.reshape(-1, ids.shape[-1]).double()
    y = torch.zeros((x2.shape[0], hidden), dtype=torch.float64, device=x.device)
    off, size = torch.zeros_like(y), torch.zeros_like(y)
    for e in range(n):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if t.numel() == 0:
            continue
        v, dv = product(x2[t], gate_up[e], gate_up_bias[e] if gate_up_bias is not None else None)
        half = v.shape[1] // 2
        a, da = activated(v[:, :half] if gated else v, dv[:, :half] if gated else dv, act)
        if gated:
            u, du = v[:, half:], dv[:, half:]
            a, da = a * u, da * (u.abs() + du) + a.abs() * du + U32 * (a * u).abs()
        h, dh = rounded(a, da)
        v, dv = product(h, down[e], down_bias[e] if down_bias is not None else None)
        dv = dv + dh @ down[e].double().abs().t()
        w = weights[t, j].unsqueeze(1)
        y.index_add_(0, t, w * v)
        off.index_add_(0, t, w.abs() * dv)
        size.index_add_(0, t, (w * v).abs())
    off = off + (ids.shape[-1] + 2) * U32 * size
    if residual is not None:
        y = y + residual.reshape(-1, hidden).double()
        off = off + U32 * y.abs()
    return y.view(x.shape), (off + U16 * (y.abs() + off)).view(x.shape)


def route(logits, top_k, scoring="softmax", bias=None, n_groups=1, top_groups=None, renormalize=True, scale=1.0):
    """route_experts in plain Python, token by token."""
    experts = logits.shape[-1]
    top_groups = n_groups if top_groups is None else top_groups
    all_ids, all_weights = [], []
    for row in logits.reshape(-1, experts).double().tolist():
        is_open = [l != -math.inf for l in row]
        if scoring == "sigmoid":
            p = [0.0 if l < -700 else 1 / (1 + math.exp(-l)) for l in row]
        else:
            most = max((l for l, o in zip(row, is_open) if o and l == l), default=0.0)
            e = [math.nan if l != l or (l == math.inf == most) else math.exp(l - most) if o else 0.0 for l, o in zip(row, is_open)]
            total = sum(e)
            p = [v / total if total else 0.0 for v in e]
        choice = list(row) if bias is None else [v + b for v, b in zip(p, bias.double().tolist())]
        choice = [math.inf if c != c else c for c in choice]
        choice = [c if o else -math.inf for c, o in zip(choice, is_open)]
        if n_groups > 1:
            size = experts // n_groups
            scores = []
            for g in range(n_groups):
                best = sorted(choice[g * size:(g + 1) * size], reverse=True)
                s = best[0]
                if bias is not None and size > 1 and best[1] != -math.inf:
                    s += best[1]
                scores.append(s)
            kept = sorted(range(n_groups), key=lambda g: (-scores[g], g))[:top_groups]
            choice = [c if i // size in kept else -math.inf for i, c in enumerate(choice)]
        order = sorted(range(experts), key=lambda i: (-choice[i], i))[:top_k]
        order = [i if choice[i] != -math.inf else -1 for i in order]
        w = [p[i] if i >= 0 else 0.0 for i in order]
        if renormalize:
            total = sum(w)
            w = [v / total if total else 0.0 for v in w]
        all_ids.append(order)
        all_weights.append([v * scale if i >= 0 else 0.0 for i, v in zip(order, w)])
    shape = logits.shape[:-1] + (top_k,)
    return torch.tensor(all_ids, dtype=torch.int32).reshape(shape), torch.tensor(all_weights, dtype=torch.float64).reshape(shape)
