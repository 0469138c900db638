"""The adapter operators (face_recognition_amd.adapter) as measured cases.

A frozen backbone answers with raw 512-wide rows; an adapter is a small residual block behind it: a norm, a dense
product with its activation, a second product back to the row's width, and a norm whose result is gated, scaled and
added to the row before it becomes a search row.  The mixture form routes every row to a few experts and takes both
products per expert.  Four operators carry it:

    linear         y = act(x W^T + b) + residual
    block_norm     out = residual + scale * g(gate) * norm(sum_j w_j x_j),   next = norm'(out)
    route          scores of logits, a bias for balance, groups, the best k, renormalised weights, rows by expert
    expert_linear  the product of every routed row with its own expert's weights

``own`` False: each operator in elementary torch operations, in 32 bits (64 where a selection stands next to a
border).  ``own`` True: the framework's kernels.
"""
import math

import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MOST_FLOPS = 2 * 16384 * 8192 * 2048


def listed():
    return [
        # one query face at serving time: the first product of an adapter behind a 512-wide backbone
        dict(name="linear one row", op="linear", type="bf16", m=1, k=512, n=2048, act="gelu", bias=True, residual=False, out="bf16"),
        # a serving batch through a wide layer: the weights are all that is read
        dict(name="linear small batch", op="linear", type="f16", m=24, k=4096, n=4096, act="relu", bias=True, residual=False, out="f16"),
        # both faces of 6000 verification pairs in the storage type of the raw embeddings
        dict(name="linear pairs f32", op="linear", type="f32", m=12000, k=512, n=512, act="prelu", bias=True, residual=True, out="f32"),
        # enrolment in bulk: the second product of a wide block, back to the row's width and onto the row
        dict(name="linear bulk", op="linear", type="bf16", m=16384, k=8192, n=2048, act="none", bias=True, residual=True, out="bf16"),
        # one row in front of the block
        dict(name="norm one row", op="block_norm", type="f32", t=1, d=512, slots=0, norm="rms", gate="none", residual=False, next="none", out="bf16"),
        # the end of a block over an enrolment chunk: gate, residual and the unit rows that search takes
        dict(name="norm to search rows", op="block_norm", type="bf16", t=65536, d=512, slots=0, norm="layer", gate="channel", residual=True, next="l2", out="bf16"),
        # the end of a mixture block: four experts' rows weighted, normed, added, and normed for the next block
        dict(name="norm of four experts", op="block_norm", type="f16", t=8191, d=2048, slots=4, norm="rms", gate="row", residual=True, next="rms", out="f32"),
        # one row picks its experts
        dict(name="route one row", op="route", type="f32", t=1, e=64, k=4, score="softmax", bias=False, groups=1, top_groups=1, padded=0),
        # a large batch picks 8 of 256 experts in 4 of 8 groups, scores biased for balance
        dict(name="route bulk", op="route", type="f32", t=65536, e=256, k=8, score="sigmoid", bias=True, groups=8, top_groups=4, padded=0),
        # a handful of rows: almost every one has experts of its own, whose weights are all that is read
        dict(name="experts small batch", op="experts", type="bf16", t=5, e=32, k=2, n=2048, d=512, act="gelu", up=True, padded=0, out="bf16"),
        # a ragged batch, padded rows at its end, back from the experts' width to slots in the rows' order
        dict(name="experts down ragged", op="experts", type="f16", t=3001, e=64, k=6, n=512, d=1536, act="none", up=False, padded=57, out="f16"),
        # bulk through the first product of 32 experts
        dict(name="experts bulk", op="experts", type="bf16", t=16384, e=32, k=4, n=4096, d=1024, act="silu", up=True, padded=0, out="bf16"),
    ]


def _log(rng, lo, hi, odd=0.5):
    """A whole number spread over the logarithm of its range; as it falls, or a multiple of 64."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() >= odd and v >= 64:
        v = v // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(["linear", "linear", "block_norm", "route", "experts", "experts"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "linear":
        while True:
            c = dict(op=op, type=kind, m=_log(rng, 1, 16384), k=_log(rng, 64, 8192, 0.25), n=_log(rng, 64, 8192, 0.25))
            if 2 * c["m"] * c["k"] * c["n"] <= MOST_FLOPS / (8 if kind == "f32" else 1):
                break
        return dict(c, act=rng.choice(["none", "prelu", "hswish", "relu", "gelu", "silu"]), bias=rng.random() < 0.8,
                    residual=rng.random() < 0.5, out=rng.choice([kind, kind, "f32"]))
    if op == "block_norm":
        while True:
            c = dict(op=op, type=kind, t=_log(rng, 1, 65536), d=_log(rng, 64, 8192, 0.25), slots=rng.choice([0, 0, 2, 4, 6]))
            if c["t"] * c["d"] * max(1, c["slots"]) <= 8191 * 2048 * 4:
                break
        return dict(c, norm=rng.choice(["rms", "layer", "none"]), gate=rng.choice(["none", "channel", "row", "full"]),
                    residual=rng.random() < 0.7, next=rng.choice(["none", "rms", "layer", "l2"]), out=rng.choice(["bf16", "f16", "f32"]))
    t = _log(rng, 1, 65536 if op == "route" else 16384)
    padded = rng.randint(0, t // 3) if rng.random() < 0.3 else 0
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        e = groups * _log(rng, 8, 256 // groups if groups > 1 else 384)
        top = rng.randint(1, groups)
        return dict(op=op, type=kind, t=t, e=e, k=rng.randint(1, min(8, top * e // groups)), score=rng.choice(["softmax", "sigmoid"]),
                    bias=rng.random() < 0.5, groups=groups, top_groups=top, padded=padded)
    while True:
        c = dict(op=op, type=kind, t=t, e=_log(rng, 4, 64), k=rng.randint(1, 4), n=_log(rng, 64, 4096, 0.25), d=_log(rng, 64, 4096, 0.25))
        if c["e"] * c["n"] * c["d"] <= 1 << 28 and 2 * t * c["k"] * c["n"] * c["d"] <= MOST_FLOPS / (8 if kind == "f32" else 4):
            break
        t = max(1, t // 2)
        padded = 0
    return dict(c, act=rng.choice(["none", "hswish", "relu", "gelu", "silu"]), up=rng.random() < 0.5, padded=min(padded, c["t"] // 3),
                out=rng.choice([kind, kind, "f32"]))


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=device).manual_seed(seed)
    dt = _TYPES[case["type"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=device) * scale).to(dtype)

    s = dict(case=case)
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"], s["w"] = normal(m, k), normal(n, k, scale=k ** -0.5)
        s["bias"] = normal(n, scale=0.5) if case["bias"] else None
        s["slope"] = 0.25 + normal(n, scale=0.05, dtype=torch.float32) if case["act"] == "prelu" else None
        s["residual"] = normal(m, n, dtype=_TYPES[case["out"]]) if case["residual"] else None
    elif case["op"] == "block_norm":
        t, d, slots = case["t"], case["d"], case["slots"]
        s["x"] = normal(t, slots, d) if slots else normal(t, d)
        s["slot_weights"] = torch.softmax(torch.randn(t, slots, generator=g, device=device), -1) if slots else None
        s["residual"] = normal(t, d, dtype=_TYPES[case["out"]]) if case["residual"] else None
        s["weight"] = 1 + normal(d, scale=0.1, dtype=torch.float32) if case["norm"] != "none" else None
        s["bias"] = normal(d, scale=0.1, dtype=torch.float32) if case["norm"] == "layer" else None
        shape = {"none": None, "channel": (d,), "row": (t, 1), "full": (t, d)}[case["gate"]]
        s["gate"] = normal(*shape) if shape else None
        s["next_weight"] = 1 + normal(d, scale=0.1, dtype=torch.float32) if case["next"] in ("rms", "layer") else None
        s["next_bias"] = normal(d, scale=0.1, dtype=torch.float32) if case["next"] == "layer" else None
    else:
        t, e = case["t"], case["e"]
        logits = torch.randn(t, e, generator=g, device=device) + 0.7 * torch.randn(e, generator=g, device=device)
        if case["padded"]:
            logits[t - case["padded"]:] = -math.inf
        logits = logits.to(dt)
        if case["op"] == "route":
            s["logits"] = logits
            s["bias"] = 0.1 * torch.randn(e, generator=g, device=device) if case["bias"] else None
            return s
        k, n, d = case["k"], case["n"], case["d"]
        top = torch.topk(logits.float(), k, dim=-1).indices
        if case["padded"]:
            top[t - case["padded"]:] = e
        flat = top.reshape(-1)
        s["order"] = torch.sort(flat, stable=True).indices.to(torch.int32)
        s["offsets"] = torch.searchsorted(torch.sort(flat).values, torch.arange(e + 1, device=device)).to(torch.int32)
        s["experts"] = torch.where(top == e, -1, top).to(torch.int32)
        s["weights"] = (torch.full((t, k), 1.0 / k, device=device) * (s["experts"] >= 0)).contiguous()
        s["x"] = normal(t if case["up"] else t * k, d)
        s["w"] = normal(e, n, d, scale=d ** -0.5)
        s["bias"] = normal(e, n, scale=0.5)
    return s


def _act(v, name, slope=None):
    if name == "prelu":
        return torch.where(v >= 0, v, v * slope)
    if name == "relu":
        return torch.clamp(v, min=0)
    if name == "hswish":
        return v * torch.clamp(v / 6 + 0.5, 0, 1)
    if name == "gelu":
        return v * 0.5 * (1 + torch.erf(v * math.sqrt(0.5)))
    if name == "silu":
        return v / (1 + torch.exp(-v))
    return v


def _norm(v, name, weight, bias):
    if name == "rms":
        return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6) * weight
    if name == "layer":
        v = v - v.mean(-1, keepdim=True)
        return v * torch.rsqrt((v * v).mean(-1, keepdim=True) + 1e-6) * weight + bias
    if name == "l2":
        return v / torch.sqrt((v * v).sum(-1, keepdim=True)).clamp_min(1e-37)
    return v


def _linear(s):
    c = s["case"]
    v = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        v = v + s["bias"].float()
    v = _act(v, c["act"], s["slope"])
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v.to(_TYPES[c["out"]])


def _block_norm(s):
    c = s["case"]
    v = s["x"].float()
    if c["slots"]:
        v = (v * s["slot_weights"][:, :, None]).sum(1)
    v = _norm(v, c["norm"], s["weight"], s["bias"])
    if s["gate"] is not None:
        v = v * s["gate"].float()
    v = v * 0.5
    if s["residual"] is not None:
        v = v + s["residual"].float()
    out = v.to(_TYPES[c["out"]])
    if c["next"] == "none":
        return out
    return out, _norm(v, c["next"], s["next_weight"], s["next_bias"]).to(torch.bfloat16)


def _route(s):
    c = s["case"]
    t, e, k, groups = c["t"], c["e"], c["k"], c["groups"]
    logits = s["logits"].double()
    scores = torch.softmax(logits, -1) if c["score"] == "softmax" else torch.sigmoid(logits)
    masked = logits == -math.inf
    # without a bias and groups the order of the scores is that of the logits
    key = scores + s["bias"].double() if s["bias"] is not None else scores if groups > 1 else logits
    key = torch.where(masked, -math.inf, key)
    if groups > 1:
        best = torch.sort(key.view(t, groups, e // groups), dim=-1, descending=True).values[:, :, :2].sum(-1)
        chosen = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :c["top_groups"]]
        keep = torch.zeros(t, groups, dtype=torch.bool, device=key.device).scatter_(1, chosen, True)
        key = torch.where(keep[:, :, None], key.view(t, groups, -1), -math.inf).view(t, e)
    best = torch.sort(key, dim=-1, descending=True, stable=True)
    experts, empty = best.indices[:, :k], best.values[:, :k] == -math.inf
    weights = torch.where(empty, 0.0, torch.gather(scores, 1, experts))
    weights = weights / weights.sum(-1, keepdim=True).clamp_min(1e-300)
    experts = torch.where(empty, -1, experts)
    flat = torch.where(empty, e, experts).reshape(-1)
    rows = torch.sort(flat, stable=True)
    offsets = torch.searchsorted(rows.values, torch.arange(e + 1, device=flat.device))
    return weights.float(), experts.to(torch.int32), rows.indices.to(torch.int32), offsets.to(torch.int32)


def _experts(s):
    """Every expert's rows side by side, padded to the longest list, in one batched product."""
    c = s["case"]
    p, offsets, order = c["t"] * c["k"], s["offsets"].long(), s["order"].long()
    at = torch.arange(p, device=order.device)
    expert = torch.searchsorted(offsets, at, right=True) - 1
    routed = expert < c["e"]
    expert = expert.clamp_max(c["e"] - 1)
    rank = torch.where(routed, at - offsets[expert], 0)
    longest = max(1, int((offsets[1:] - offsets[:-1]).max()))
    x = s["x"].float()[order // c["k"]] if c["up"] else s["x"].float()
    beside = torch.zeros(c["e"], longest, c["d"], device=x.device)
    beside[expert[routed], rank[routed]] = x[routed]
    v = torch.bmm(beside, s["w"].float().transpose(1, 2).contiguous()) + s["bias"].float()[:, None, :]
    v = torch.where(routed[:, None], _act(v, c["act"])[expert, rank], 0.0).to(_TYPES[c["out"]])
    if c["up"]:
        return v
    out = torch.empty_like(v)
    out[order] = v
    return out.view(c["t"], c["k"], c["n"])


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"linear": _linear, "block_norm": _block_norm, "route": _route, "experts": _experts}[c["op"]](s)
    from face_recognition_amd import adapter
    if c["op"] == "linear":
        return adapter.linear(s["x"], s["w"], s["bias"], act=c["act"], slope=s["slope"], residual=s["residual"], out_dtype=_TYPES[c["out"]])
    if c["op"] == "block_norm":
        more = {} if c["next"] == "none" else dict(next_norm=c["next"], next_weight=s["next_weight"], next_bias=s["next_bias"],
                                                   next_dtype=torch.bfloat16)
        return adapter.block_norm(s["x"], s["residual"], slot_weights=s["slot_weights"], norm=c["norm"], weight=s["weight"],
                                  bias=s["bias"], gate=s["gate"], scale=0.5, out_dtype=_TYPES[c["out"]], **more)
    if c["op"] == "route":
        return tuple(adapter.route(s["logits"], c["k"], score=c["score"], bias=s["bias"], groups=c["groups"], top_groups=c["top_groups"]))
    routing = adapter.Routing(s["weights"], s["experts"], s["order"], s["offsets"])
    return adapter.expert_linear(s["x"], s["w"], routing, s["bias"], act=c["act"], rows="tokens" if c["up"] else "sorted",
                                 out="sorted" if c["up"] else "slots", out_dtype=_TYPES[c["out"]])


def work(case):
    size = {k: v.itemsize for k, v in _TYPES.items()}
    b = size[case["type"]]
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        o = size[case["out"]]
        return {"bytes": (m * k + n * k + n * case["bias"]) * b + m * n * o * (2 if case["residual"] else 1), "flops": 2 * m * k * n}
    if case["op"] == "block_norm":
        t, d, slots = case["t"], case["d"], case["slots"]
        gate = {"none": 0, "channel": d, "row": t, "full": t * d}[case["gate"]]
        o = size[case["out"]]
        nbytes = t * d * max(1, slots) * b + 4 * t * slots + gate * b + t * d * o * (2 if case["residual"] else 1) + (0 if case["next"] == "none" else 2 * t * d)
        return {"bytes": nbytes, "flops": t * d * (2 * slots + 12)}
    t, e, k = case["t"], case["e"], case["k"]
    if case["op"] == "route":
        return {"bytes": t * e * b + t * k * 12 + 4 * (e + 1), "flops": t * e * 8}
    live, n, d = (t - case["padded"]) * k, case["n"], case["d"]
    used = e * (1 - (1 - 1 / e) ** live)  # experts that have a row, as expected of even routing
    rows = (t if case["up"] else t * k) * d
    return {"bytes": (rows + used * n * (d + 1)) * b + t * k * n * size[case["out"]] + 4 * t * k, "flops": 2 * live * n * d}


# ---- the definitions in 64 bits ---------------------------------------------------------------------------------------

def _act64(v, name, slope):
    if name == "prelu":
        return v.clamp_min(0) + slope.double() * v.clamp_max(0)
    if name == "hswish":
        return v * (v + 3).clamp(0, 6) / 6
    if name == "relu":
        return v.clamp_min(0)
    if name == "gelu":
        return 0.5 * v * torch.special.erfc(-v / math.sqrt(2.0))
    if name == "silu":
        return v * torch.special.expit(v)
    return v


def _norm64(v, name, weight, bias):
    if name == "none":
        return v
    if name == "l2":
        return v / torch.linalg.vector_norm(v, dim=-1, keepdim=True).clamp_min(1e-37)
    if name == "layer":
        var, mean = torch.var_mean(v, dim=-1, keepdim=True, correction=0)
        return (v - mean) / torch.sqrt(var + 1e-6) * weight.double() + bias.double()
    return v / torch.sqrt(torch.linalg.vector_norm(v, dim=-1, keepdim=True) ** 2 / v.shape[-1] + 1e-6) * weight.double()


def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "linear":
        v = torch.nn.functional.linear(s["x"].double(), s["w"].double(), None if s["bias"] is None else s["bias"].double())
        v = _act64(v, c["act"], s["slope"])
        return v if s["residual"] is None else v + s["residual"].double()
    if c["op"] == "block_norm":
        v = s["x"].double()
        if c["slots"]:
            v = torch.matmul(s["slot_weights"].double()[:, None, :], v)[:, 0]
        v = 0.5 * _norm64(v, c["norm"], s["weight"], s["bias"]) * (1.0 if s["gate"] is None else s["gate"].double())
        if s["residual"] is not None:
            v = s["residual"].double() + v
        return v if c["next"] == "none" else (v, _norm64(v, c["next"], s["next_weight"], s["next_bias"]))
    if c["op"] == "route":
        logits = s["logits"].double()
        if c["score"] == "softmax":
            p = torch.exp(logits - logits.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
        else:
            p = torch.special.expit(logits)
        key = p if s["bias"] is None else p + s["bias"].double()
        key = key.masked_fill(torch.isneginf(logits), -math.inf)
        if c["groups"] > 1:
            by = key.unflatten(-1, (c["groups"], -1))
            rank = torch.argsort(torch.argsort(-by.topk(2, -1).values.sum(-1), dim=-1, stable=True), dim=-1)
            key = by.masked_fill((rank >= c["top_groups"])[..., None], -math.inf).flatten(1)
        live = torch.isfinite(key)
        top = key.topk(c["k"], -1)
        w = p.gather(1, top.indices) * live.gather(1, top.indices)
        return torch.nan_to_num(w / w.sum(-1, keepdim=True)), None, None, None
    x, w, order = s["x"].double(), s["w"], s["order"].long()
    out = torch.zeros(c["t"] * c["k"], c["n"], dtype=torch.float64, device=x.device)
    edge = s["offsets"].tolist()
    for e in range(c["e"]):
        at = order[edge[e]:edge[e + 1]]
        rows = x[at // c["k"]] if c["up"] else x[edge[e]:edge[e + 1]]
        v = _act64(rows @ w[e].double().T + s["bias"][e].double(), c["act"], None)
        if c["up"]:
            out[edge[e]:edge[e + 1]] = v
        else:
            out[at] = v
    return out if c["up"] else out.view(c["t"], c["k"], c["n"])
