"""The adapter operators by their definitions, in 64 bits on any device (test infrastructure)."""
import math

import torch


def act(v, name, slope=None):
    v = v.double()
    if name == "prelu":
        return torch.where(v >= 0, v, v * slope.double())
    if name == "relu":
        return v.clamp_min(0)
    if name == "hswish":
        return v * (v / 6 + 0.5).clamp(0, 1)
    if name == "hsigmoid":
        return (v / 6 + 0.5).clamp(0, 1)
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v * math.sqrt(0.5))
    if name == "silu":
        return v * torch.sigmoid(v)
    assert name == "none"
    return v


def linear(x, w, bias=None, slope=None, residual=None, name="none"):
    v = x.double() @ w.double().T
    if bias is not None:
        v = v + bias.double()
    v = act(v, name, slope)
    return v if residual is None else v + residual.double()


def norm(y, name, weight=None, bias=None, eps=1e-6):
    if name == "none":
        return y
    if name == "l2":
        n = y.pow(2).sum(-1, keepdim=True).sqrt()
        return torch.where(n == 0, torch.zeros_like(y), y / n)
    if name == "layer":
        y = y - y.mean(-1, keepdim=True)
    y = y / (y.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        y = y * weight.double()
    return y if bias is None else y + bias.double()


def weighted(x, slot_weights):
    x = torch.where(slot_weights[..., None] == 0, torch.zeros((), dtype=torch.float64, device=x.device), x.double())
    return (x * slot_weights.double()[..., None]).sum(-2)


def gate_of(gate, name):
    g = gate.double()
    return torch.sigmoid(g) if name == "sigmoid" else torch.tanh(g) if name == "tanh" else g


def route(logits, k, score="softmax", bias=None, groups=1, top_groups=1, renormalise=True, scale=1.0):
    """Row by row in Python numbers: (weights, experts, order, offsets)."""
    T, E = logits.shape
    rows = logits.double().cpu().tolist()
    b = [0.0] * E if bias is None else bias.double().cpu().tolist()
    weights, experts = [], []
    for row in rows:
        seen = [not math.isnan(v) and v > -math.inf for v in row]
        live = [s and not math.isnan(c) and c > -math.inf for s, c in zip(seen, b)]
        top = max([v for v, s in zip(row, seen) if s], default=0.0)
        e = [(1.0 if v == top else math.exp(v - top)) if s else 0.0 for v, s in zip(row, seen)]
        z = sum(e)
        if score == "softmax":
            p = [v / z if s else 0.0 for v, s in zip(e, seen)]
        else:
            p = [(1 / (1 + math.exp(-v)) if v >= 0 else math.exp(v) / (1 + math.exp(v))) if s else 0.0 for v, s in zip(row, seen)]
        plain = bias is None and groups == 1
        key = [(v if plain else q + c) if l else -math.inf for v, q, c, l in zip(row, p, b, live)]
        if groups > 1:
            per = E // groups
            two = [sorted(key[g * per:(g + 1) * per])[-2:] for g in range(groups)]
            best = [sum(v) if v[0] > -math.inf else -math.inf for v in two]      # of a lone expert too, whatever its bias
            keep = sorted(range(groups), key=lambda g: (-best[g], g))[:top_groups]
            key = [v if i // per in keep else -math.inf for i, v in enumerate(key)]
        pick = [i for i in sorted(range(E), key=lambda i: (-key[i], i))[:k] if key[i] > -math.inf]
        if renormalise and pick:
            # as ratios to the greatest, so that scores too small for a double still have them
            if score == "softmax" or max(row[i] for i in pick) < -30:
                m = max(row[i] for i in pick)
                w = [1.0 if row[i] == m else math.exp(row[i] - m) for i in pick]
            else:
                w = [p[i] for i in pick]
            w = [v / sum(w) for v in w]
        else:
            w = [p[i] for i in pick]
        weights.append([v * scale for v in w] + [0.0] * (k - len(pick)))
        experts.append(pick + [-1] * (k - len(pick)))
    flat = [E if e < 0 else e for r in experts for e in r]
    order = sorted(range(T * k), key=lambda s: flat[s])
    offsets = [sum(1 for e in flat if e < i) for i in range(E + 1)] if T * k < 100000 else None
    return (torch.tensor(weights, dtype=torch.float64).reshape(T, k), torch.tensor(experts, dtype=torch.int32).reshape(T, k),
            torch.tensor(order, dtype=torch.int32), torch.tensor(offsets, dtype=torch.int32))


def routing_of(experts, E):
    """(order, offsets) of a given choice [T, k] (-1: none)."""
    flat = torch.where(experts < 0, E, experts.long()).reshape(-1).cpu()
    order = torch.sort(flat, stable=True).indices.to(torch.int32)
    offsets = torch.tensor([(flat < e).sum() for e in range(E + 1)], dtype=torch.int32)
    return order.to(experts.device), offsets.to(experts.device)


def expert_linear(x, w, experts, bias=None, slope=None, name="none", tokens=True, slots=False):
    """x [T, K] or, tokens False, [T * k, K] in the order's positions -> [T * k, N] by position, or [T, k, N]."""
    T, k = experts.shape
    E, N, _ = w.shape
    order, _ = routing_of(experts, E)
    flat = experts.reshape(-1).tolist()
    out = torch.zeros(T * k, N, dtype=torch.float64, device=x.device)
    for p, s in enumerate(order.tolist()):
        e = flat[s]
        if e >= 0:
            row = x[s // k] if tokens else x[p]
            out[s if slots else p] = linear(row[None], w[e], None if bias is None else bias[e], None if slope is None else slope[e], None, name)[0]
    return out.view(T, k, N) if slots else out
