"""Adapter blocks between a backbone and the search (no counterpart in the reference).

A frozen backbone answers with raw rows (inference.py:121-122); an adapter fitted elsewhere -- to a camera, to masked
faces, to a new domain -- is a residual block over those rows.  This module holds the block's operators and the two
blocks made of them:

    linear         act(x W^T + b) + residual
    block_norm     out = residual + scale * g(gate) * norm(y), next = norm'(out); y = x or a weighted sum of expert rows
    route          scores of logits -> the best k experts of every row, their weights, and the slots sorted by expert
    expert_linear  every routed row times its own expert's weights

    ResidualAdapter   rows -> norm -> linear, act -> linear -> norm, gate, scale, + rows
    ExpertAdapter     the same with both products per expert

``adapter(emb)`` gives adapted embeddings, ``adapter.rows(emb)`` the L2-normalised bf16 rows that ``search.Matcher`` and
``gallery.GalleryWriter.add_normalized`` take.  Inference only, as everything here: tensors that ask for a gradient are
refused.  All four operators are ``torch.ops.fr_hip`` ops over the C ABI (include/fr_hip.h), run on the current stream of
their tensors' device, allocate with torch's caching allocator, synchronise nothing and can be captured into a graph.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import ops as _ops


_DIRECT = {"linear": _ops._linear, "block_norm": _ops._block_norm_eager, "route": _ops._route, "expert_linear": _ops._expert_linear}


def _op(name: str, x: torch.Tensor):
    """The operator for a call on ``x``: its implementation itself for an eager call on plain tensors (the dispatcher takes
    as long as the smallest kernels run), ``torch.ops.fr_hip`` for whatever traces or stands in for one.  The first look is at
    ``x``; what the other arguments hold is seen by the implementation, which turns to ``torch.ops.fr_hip`` too."""
    kind = type(x)
    if (kind is torch.Tensor or kind is torch.nn.Parameter) and not torch.compiler.is_compiling():
        return _DIRECT[name]
    return getattr(torch.ops.fr_hip, name)


def _need_gpu(x: torch.Tensor, what: str) -> None:
    if not x.is_cuda:
        raise RuntimeError(f"{what} needs GPU tensors: the hot path has no CPU fallback")


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, act: str = "none",
           slope: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None,
           out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``: x [..., K], weight [N, K] of one type (bf16, f16, f32), bias [N] of that
    type or f32, residual [..., N] of any of the three.  act: none, prelu (slope f32 [N]), hswish, relu, hsigmoid, gelu
    (erf form), silu.  Accumulation and epilogue in f32, rounded once to ``out_dtype`` (x's type by default)."""
    _need_gpu(x, "linear")
    return _op("linear", x)(x, weight, bias, slope, residual, act, out_dtype)


def block_norm(x: torch.Tensor, residual: Optional[torch.Tensor] = None, *, slot_weights: Optional[torch.Tensor] = None,
               norm: str = "rms", weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, eps: float = 1e-6,
               gate: Optional[torch.Tensor] = None, gate_act: str = "none", scale: float = 1.0,
               next_norm: Optional[str] = None, next_weight: Optional[torch.Tensor] = None,
               next_bias: Optional[torch.Tensor] = None, next_eps: float = 1e-6, out_dtype: Optional[torch.dtype] = None,
               next_dtype: Optional[torch.dtype] = None) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``out = residual + scale * g(gate) * norm(y)`` for x [..., d], and with ``next_norm`` also ``next = next_norm(out)``
    of the unrounded out.  y is x, or with slot_weights f32 [..., S] the sum of ``slot_weights[..., j] * x[..., j, :]`` over
    x [..., S, d] (a slot of weight 0 is skipped, whatever it holds).  Norms: none, rms, layer, l2 (a zero row stays zero);
    weight / bias f32 [d] for rms and layer.  gate: [d], [..., 1] or [..., d]; gate_act none, sigmoid, tanh.  d <= 16384.
    Returns out, or (out, next)."""
    _need_gpu(x, "block_norm")
    out, nxt = _op("block_norm", x)(x, residual, slot_weights, norm, weight, bias, eps, gate, gate_act, scale,
                                           next_norm or "none", next_weight, next_bias, next_eps, out_dtype, next_dtype)
    return (out, nxt) if next_norm not in (None, "none") else out


class Routing(NamedTuple):
    """What ``route`` answers for T rows: slot ``t * k + j`` is row t's j-th choice."""
    weights: torch.Tensor      # f32 [T, k], 0 where there is no expert
    experts: torch.Tensor      # int32 [T, k], best first, -1 where there is none
    order: torch.Tensor        # int32 [T * k]: slots sorted by expert, stable; those without an expert last
    offsets: torch.Tensor      # int32 [E + 1]: expert e's slots are order[offsets[e]:offsets[e + 1]]


def route(logits: torch.Tensor, k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None, groups: int = 1,
          top_groups: int = 1, renormalise: bool = True, scale: float = 1.0) -> Routing:
    """The k experts of every row of logits [T, E].  Scores are a softmax over the row or sigmoids; ``bias`` f32 [E] moves
    the choice but not the weights; ``groups`` equal runs of experts limit it to the ``top_groups`` runs whose best two
    biased scores add up to most.  Ties go to the lower index.  weights: the chosen scores, over their sum if
    ``renormalise``, times ``scale``.  Logits (or biases) that are -inf or NaN mask their expert; a row whose mask leaves
    fewer than k has slots of expert -1 and weight 0.  E <= 512, k <= 16, groups <= 64."""
    _need_gpu(logits, "route")
    return Routing(*_op("route", logits)(logits, k, score, bias, groups, top_groups, renormalise, scale))


def expert_linear(x: torch.Tensor, weight: torch.Tensor, routing: Routing, bias: Optional[torch.Tensor] = None, *,
                  act: str = "none", slope: Optional[torch.Tensor] = None, rows: str = "tokens", out: str = "sorted",
                  out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """``act(row @ weight[e].T + bias[e])`` for every slot of ``routing``: weight [E, N, K], bias [E, N].  rows="tokens"
    takes x [T, K] (each row once per expert it chose), rows="sorted" x [T * k, K] in the order's positions;
    out="sorted" answers [T * k, N] in those positions, out="slots" [T, k, N] by slot, ready for ``block_norm``'s
    slot_weights.  Slots without an expert get zero rows.  The tables are taken as ``route`` gives them: nothing is written
    for an entry of the order that names no slot."""
    _need_gpu(x, "expert_linear")
    return _op("expert_linear", x)(x, weight, routing.order, routing.offsets, routing.experts.shape[1], bias, act, slope,
                                          rows, out, out_dtype)


class _Block(torch.nn.Module):
    """Norms, gate and the two ends that both blocks share."""

    def __init__(self, dim: int, norm: str, act: str, scale: float, dtype: torch.dtype) -> None:
        super().__init__()
        if norm not in ("rms", "layer"):
            raise ValueError(f"norm is 'rms' or 'layer': got {norm!r}")
        if act == "prelu" or act not in _ops._ACTS:
            raise ValueError(f"act is one of {', '.join(a for a in _ops._ACTS if a != 'prelu')}: got {act!r}")
        if dtype not in _ops._TYPES:
            raise ValueError(f"dtype is float32, bfloat16 or float16: got {dtype}")
        self.dim, self.norm, self.act, self.scale, self.dtype = dim, norm, act, scale, dtype
        self._add("pre_weight", torch.ones(dim))
        self._add("post_weight", torch.ones(dim))
        if norm == "layer":
            self._add("pre_bias", torch.zeros(dim))
            self._add("post_bias", torch.zeros(dim))
        else:
            self.pre_bias = self.post_bias = None
        self._add("gate", torch.zeros(dim))                   # a block that was given no weights changes nothing

    def _add(self, name: str, value: torch.Tensor) -> None:
        self.register_parameter(name, torch.nn.Parameter(value, requires_grad=False))

    def _matrix(self, name: str, *shape: int) -> None:
        self._add(name, (torch.randn(*shape) * shape[-1] ** -0.5).to(self.dtype))

    def _check(self, x: torch.Tensor) -> None:
        _need_gpu(x, type(self).__name__)
        if x.dim() != 2 or x.shape[1] != self.dim:
            raise ValueError(f"expected [n, {self.dim}] rows, got {tuple(x.shape)}")

    def _pre(self, x: torch.Tensor) -> torch.Tensor:
        return block_norm(x, norm=self.norm, weight=self.pre_weight, bias=self.pre_bias, out_dtype=self.dtype)

    def _post(self, y: torch.Tensor, x: torch.Tensor, slot_weights: Optional[torch.Tensor], **more):
        return block_norm(y, x, slot_weights=slot_weights, norm=self.norm, weight=self.post_weight, bias=self.post_bias,
                          gate=self.gate, scale=self.scale, out_dtype=x.dtype, **more)

    def _branch(self, x: torch.Tensor) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        raise NotImplementedError

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        """Rows [n, dim] (what a backbone returns) -> adapted rows of the same type."""
        self._check(x)
        y, slot_weights = self._branch(x)
        return self._post(y, x, slot_weights)

    def rows(self, x: torch.Tensor) -> torch.Tensor:
        """Rows [n, dim] -> adapted, L2-normalised bf16 rows: gallery and query format of the search."""
        self._check(x)
        y, slot_weights = self._branch(x)
        return self._post(y, x, slot_weights, next_norm="l2", next_dtype=torch.bfloat16)[1]


class ResidualAdapter(_Block):
    """x + scale * gate * norm(W2 act(W1 norm(x) + b1) + b2)."""

    def __init__(self, dim: int = 512, hidden: int = 2048, *, norm: str = "layer", act: str = "gelu", scale: float = 1.0,
                 dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__(dim, norm, act, scale, dtype)
        self._matrix("w1", hidden, dim)
        self._matrix("w2", dim, hidden)
        self._add("b1", torch.zeros(hidden, dtype=dtype))
        self._add("b2", torch.zeros(dim, dtype=dtype))

    def _branch(self, x):
        return linear(linear(self._pre(x), self.w1, self.b1, act=self.act), self.w2, self.b2), None


class ExpertAdapter(_Block):
    """x + scale * gate * norm(sum_j w_j (W2_e(j) act(W1_e(j) norm(x) + b1_e(j)) + b2_e(j))), the k experts of a row by a
    router over norm(x)."""

    def __init__(self, dim: int = 512, hidden: int = 2048, experts: int = 8, k: int = 2, *, norm: str = "layer", act: str = "gelu",
                 scale: float = 1.0, score: str = "softmax", groups: int = 1, top_groups: int = 1,
                 dtype: torch.dtype = torch.bfloat16) -> None:
        super().__init__(dim, norm, act, scale, dtype)
        self.k, self.score, self.groups, self.top_groups = k, score, groups, top_groups
        self._matrix("router", experts, dim)
        self._add("balance", torch.zeros(experts))
        self._matrix("w1", experts, hidden, dim)
        self._matrix("w2", experts, dim, hidden)
        self._add("b1", torch.zeros(experts, hidden, dtype=dtype))
        self._add("b2", torch.zeros(experts, dim, dtype=dtype))

    def _branch(self, x):
        h = self._pre(x)
        r = route(linear(h, self.router, out_dtype=torch.float32), self.k, score=self.score, bias=self.balance, groups=self.groups,
                  top_groups=self.top_groups)
        up = expert_linear(h, self.w1, r, self.b1, act=self.act)
        return expert_linear(up, self.w2, r, self.b2, rows="sorted", out="slots"), r.weights
