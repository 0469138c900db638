"""Adapter operators and torch's dispatcher: what a tensor or a thread carries besides memory (a negative bit, a subclass, a
tracer, a mode, a transform, a gradient) is not lost by the short way that plain calls take."""
import pytest
import torch

from face_recognition_amd import _lib, adapter, ops
from test_adapter import gen, randn

OPS = ("linear", "block_norm", "route", "expert_linear")


def arguments(device, seed=1):
    """Positional arguments of the four operators, every optional tensor given."""
    g = gen(seed, device)
    x, w, b, slope, res = randn(g, 6, 16), randn(g, 12, 16), randn(g, 12), randn(g, 12), randn(g, 6, 12)
    y, sw, v = randn(g, 6, 2, 16), torch.rand(6, 2, generator=g, device=device), [randn(g, 16) for _ in range(4)]
    logits, lb = randn(g, 6, 8), randn(g, 8, scale=0.1)
    order, offsets = torch.arange(12, dtype=torch.int32, device=device), torch.tensor([0, 5, 5, 12], dtype=torch.int32, device=device)
    we, be, se = randn(g, 3, 12, 16), randn(g, 3, 12), randn(g, 3, 12)
    return {"linear": (x, w, b, slope, res, "prelu", None),
            "block_norm": (y, randn(g, 6, 16), sw, "layer", v[0], v[1], 1e-6, randn(g, 6, 1), "tanh", 0.5, "layer", v[2], v[3], 1e-6, None, None),
            "route": (logits, 2, "sigmoid", lb, 2, 1, True, 1.0),
            "expert_linear": (x, we, order, offsets, 2, be, "prelu", se, "tokens", "slots", None)}


def function(name, args):
    """The public function of ``adapter`` on an operator's positional arguments."""
    if name == "linear":
        x, w, b, slope, res, act, out = args
        return adapter.linear(x, w, b, act=act, slope=slope, residual=res, out_dtype=out)
    if name == "block_norm":
        x, res, sw, norm, w, b, eps, gate, ga, scale, nn, nw, nb, ne, od, nd = args
        return adapter.block_norm(x, res, slot_weights=sw, norm=norm, weight=w, bias=b, eps=eps, gate=gate, gate_act=ga, scale=scale,
                                  next_norm=nn, next_weight=nw, next_bias=nb, next_eps=ne, out_dtype=od, next_dtype=nd)
    if name == "route":
        logits, k, score, b, groups, top, again, scale = args
        return tuple(adapter.route(logits, k, score=score, bias=b, groups=groups, top_groups=top, renormalise=again, scale=scale))
    x, w, order, offsets, k, b, act, slope, rows, out, od = args
    experts = torch.zeros(order.numel() // k, k, dtype=torch.int32, device=order.device)
    return adapter.expert_linear(x, w, adapter.Routing(experts.float(), experts, order, offsets), b, act=act, slope=slope, rows=rows, out=out, out_dtype=od)


def tensors(args):
    return [i for i, a in enumerate(args) if isinstance(a, torch.Tensor)]


def replaced(args, i, value):
    return args[:i] + (value,) + args[i + 1:]


def flat(v):
    return tuple(v) if isinstance(v, tuple) else (v,)


def same(got, want, what=""):
    got, want = flat(got), flat(want)
    assert len(got) == len(want), what
    for a, b in zip(got, want):
        assert a.dtype == b.dtype and torch.equal(a, b), what


CODES = {"linear": {5: 1}, "block_norm": {3: 2, 8: 2, 10: 2}, "route": {2: 1}, "expert_linear": {6: 1, 8: 0, 9: 1}}


def short(name, args):
    """The compiled way's answer: on CPU tensors None, or NotImplemented where the dispatcher has something to do."""
    args = tuple(CODES[name].get(i, a) for i, a in enumerate(args))
    return getattr(_lib.calls(), name)(*args, 0, 0)


class Seen(torch.Tensor):
    """A subclass that notes which operators it meets."""
    met = []

    @classmethod
    def __torch_function__(cls, func, types, args=(), kwargs=None):
        cls.met.append(str(func))
        with torch._C.DisableTorchFunctionSubclass():
            return func(*args, **(kwargs or {}))


# ---- tensors that are more than memory ---------------------------------------------------------------------------------

@pytest.mark.parametrize("name", OPS)
def test_short_way_leaves_such_tensors_to_the_dispatcher(name):
    args = arguments("cpu")[name]
    assert short(name, args) is None                           # a plain call, though not one for the GPU
    for i in tensors(args):
        assert short(name, replaced(args, i, torch._neg_view(args[i]))) is NotImplemented, i
        assert short(name, replaced(args, i, args[i].as_subclass(Seen))) is NotImplemented, i
        assert short(name, replaced(args, i, torch.nn.Parameter(args[i], requires_grad=False))) is None, i
    assert short(name, replaced(args, 0, torch._efficientzerotensor(args[0].shape))) is NotImplemented


@pytest.mark.gpu
@pytest.mark.parametrize("name", OPS)
def test_negative_bit(name):
    args = arguments("cuda")[name]
    want = function(name, args)
    for i in tensors(args):
        if args[i].is_floating_point():
            lazy = torch._neg_view(-args[i])
            assert lazy.is_neg() and lazy.is_contiguous() and torch.equal(lazy, args[i])
            same(function(name, replaced(args, i, lazy)), want, (name, i))
            same(getattr(torch.ops.fr_hip, name)(*replaced(args, i, lazy)), want, (name, i))


@pytest.mark.gpu
def test_negative_bit_of_a_conjugate():
    z = torch.tensor([[1 + 2j], [3 - 4j]], device="cuda").conj().imag
    assert z.is_neg() and z.stride() == (2, 2)                 # rows apart, taken as they lie
    assert adapter.linear(z, torch.ones(1, 1, device="cuda")).tolist() == [[-2.0], [4.0]]


@pytest.mark.gpu
@pytest.mark.parametrize("name", OPS)
def test_subclass_in_any_place(name):
    args = arguments("cuda")[name]
    want = function(name, args)
    for i in tensors(args):
        Seen.met.clear()
        got = function(name, replaced(args, i, args[i].as_subclass(Seen)))
        assert any("fr_hip" in f and name in f for f in Seen.met), (name, i, Seen.met)
        same(tuple(t.as_subclass(torch.Tensor) for t in flat(got)), want, (name, i))
