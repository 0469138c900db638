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


# ---- threads in a tracer, a mode or a transform ------------------------------------------------------------------------

class Counting(torch.utils._python_dispatch.TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.met = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.met.append(str(func))
        return func(*args, **(kwargs or {}))


class CountingFunctions(torch.overrides.TorchFunctionMode):
    def __init__(self):
        super().__init__()
        self.met = []

    def __torch_function__(self, func, types, args=(), kwargs=None):
        self.met.append(str(func))
        return func(*args, **(kwargs or {}))


def traced(name, args, run):
    """``run`` on ``name`` as a function of its first argument, as make_fx and jit.trace take it."""
    return lambda x: run(name, (x,) + args[1:])


@pytest.mark.parametrize("name", OPS)
def test_short_way_leaves_such_threads_to_the_dispatcher(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    args = arguments("cpu")[name]
    said = []

    def ask(x):
        said.append(short(name, (x,) + args[1:]))
        return x + 1

    ask(args[0])
    with torch.no_grad(), torch.autocast("cpu"):
        ask(args[0])
    with torch.inference_mode():
        ask(args[0])
    assert said == [None] * 3
    said.clear()
    for run in (lambda: make_fx(ask)(args[0]), lambda: torch.jit.trace(ask, args[0], check_trace=False), lambda: torch.func.vmap(ask)(args[0][None]),
                lambda: torch.func.jvp(ask, (args[0],), (args[0],)), lambda: torch.func.grad(lambda x: ask(x).sum())(args[0])):
        run()
        assert said and all(a is NotImplemented for a in said), said
        said.clear()
    for mode in (Counting(), CountingFunctions()):
        with mode:
            ask(args[0])
        assert said.pop() is NotImplemented
    ask(args[0])
    assert said == [None]                                      # and nothing of it stays behind


@pytest.mark.gpu
@pytest.mark.parametrize("name", OPS)
def test_tracers_record_the_operator(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    args, other = arguments("cuda")[name], arguments("cuda", 2)[name]
    graph = make_fx(traced(name, args, function))(args[0])
    assert any(f"fr_hip.{name}" in str(n.target) for n in graph.graph.nodes), graph.code
    want = function(name, (other[0],) + args[1:])
    same(graph(other[0]), want, name)
    for kind in ("fake", "symbolic"):
        graph = make_fx(traced(name, args, function), tracing_mode=kind, _allow_non_fake_inputs=True)(args[0])
        assert any(f"fr_hip.{name}" in str(n.target) for n in graph.graph.nodes), graph.code
        same(graph(other[0]), want, (name, kind))
    script = torch.jit.trace(traced(name, args, function), args[0])
    assert f"fr_hip::{name}" in str(script.graph)
    same(script(other[0]), want, name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", OPS)
def test_modes_see_the_operator(name):
    args = arguments("cuda")[name]
    want = function(name, args)
    for mode in (Counting(), CountingFunctions()):
        with mode:
            got = function(name, args)
        assert any("fr_hip" in f and name in f for f in mode.met), mode.met
        same(got, want, name)


@pytest.mark.gpu
def test_maps_over_a_batch():
    x, w = randn(gen(3), 5, 6, 16), randn(gen(4), 12, 16)
    assert torch.equal(torch.func.vmap(lambda r: adapter.linear(r, w))(x), torch.stack([adapter.linear(r, w) for r in x]))
    assert torch.equal(torch.func.vmap(adapter.block_norm)(x), torch.stack([adapter.block_norm(r) for r in x]))


@pytest.mark.gpu
@pytest.mark.parametrize("name", OPS)
def test_compiled_programs_hold_the_operator(name):
    args, other = arguments("cuda")[name], arguments("cuda", 2)[name]
    graphs = []

    def backend(graph, inputs):
        graphs.append(graph)
        return graph.forward

    torch._dynamo.reset()
    compiled = torch.compile(traced(name, args, function), backend=backend, fullgraph=True)
    same(compiled(other[0]), function(name, (other[0],) + args[1:]), name)
    assert any(f"fr_hip.{name}" in str(n.target) for n in graphs[0].graph.nodes), graphs[0].code
    torch._dynamo.reset()


# ---- gradients ---------------------------------------------------------------------------------------------------------

def refused(call, words):
    with pytest.raises(RuntimeError, match="inference only") as e:
        call()
    assert words in str(e.value)


def refuses_gradients(name, args, call):
    """``call(args)`` says no to a gradient or a tangent of any of its tensors, by whatever way it is asked for."""
    from torch.autograd import forward_ad
    for i in tensors(args):
        t = args[i]
        if not t.is_floating_point():
            continue
        one = lambda v, i=i: call(replaced(args, i, v))
        refused(lambda: one(t.clone().requires_grad_()), "no_grad")
        with torch.no_grad():
            assert not any(y.requires_grad for y in flat(one(t.clone().requires_grad_())))
        with forward_ad.dual_level():
            refused(lambda: one(forward_ad.make_dual(t, torch.ones_like(t))), "tangent")
            with torch.no_grad():                              # which does not turn these off
                refused(lambda: one(forward_ad.make_dual(t, torch.ones_like(t))), "tangent")
            one(t)                                             # another's level is no reason
        refused(lambda: torch.func.jvp(one, (t,), (torch.ones_like(t),)), "tangent")
        refused(lambda: torch.func.vjp(one, t), "no_grad")
        refused(lambda: torch.func.grad(lambda v: flat(one(v))[0].sum())(t), "no_grad")


@pytest.mark.parametrize("name", OPS)
def test_dispatched_gradients_are_refused(name):
    """Through the dispatcher, on tensors without data."""
    args = tuple(a.to("meta") if isinstance(a, torch.Tensor) else a for a in arguments("cpu")[name])
    refuses_gradients(name, args, lambda a: getattr(torch.ops.fr_hip, name)(*a))


@pytest.mark.parametrize("name", OPS)
def test_direct_tangents_are_refused(name):
    from torch.autograd import forward_ad
    args = arguments("cpu")[name]
    impl = {"linear": ops._linear, "block_norm": ops._block_norm, "route": ops._route, "expert_linear": ops._expert_linear}[name]
    with forward_ad.dual_level():
        for i in tensors(args):
            if args[i].is_floating_point():
                refused(lambda: impl(*replaced(args, i, forward_ad.make_dual(args[i], args[i]))), "tangent")


@pytest.mark.gpu
@pytest.mark.parametrize("name", OPS)
def test_gradients_and_tangents_are_refused_on_the_gpu(name):
    args = arguments("cuda")[name]
    refuses_gradients(name, args, lambda a: function(name, a))
    refuses_gradients(name, args, lambda a: getattr(torch.ops.fr_hip, name)(*a))


@pytest.mark.parametrize("name", OPS)
def test_fake_tensors_need_no_gpu(name):
    """Shapes of GPU tensors that only stand in for some, through the functions and the dispatched operators."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    real = arguments("cpu")[name]
    with FakeTensorMode():
        args = tuple(torch.empty(a.shape, dtype=a.dtype, device="cuda") if isinstance(a, torch.Tensor) else a for a in real)
        for got in (function(name, args), getattr(torch.ops.fr_hip, name)(*args)):
            assert all(y.is_cuda for y in flat(got))
        refused(lambda: getattr(torch.ops.fr_hip, name)(*replaced(args, 0, args[0].requires_grad_())), "no_grad")


# ---- tensors without data ----------------------------------------------------------------------------------------------

def refusals():
    """Every refusal that the functions are tested for, and some that stand in the C entries."""
    import test_adapter as ta
    base = {"linear": dict(x=torch.zeros(2, 8), weight=torch.zeros(4, 8), **ta.LINEAR), "block_norm": dict(x=torch.zeros(2, 8), **ta.NORM),
            "route": dict(logits=torch.zeros(2, 8), **ta.ROUTE), "expert_linear": dict(x=torch.zeros(2, 8), weight=torch.zeros(3, 4, 8), **ta.EXPERT)}
    for name, test in zip(OPS, (ta.test_linear_refuses, ta.test_block_norm_refuses, ta.test_route_refuses, ta.test_expert_linear_refuses)):
        for change, words in test.pytestmark[0].args[1]:
            if words != "all tensors on":                      # all of these are on one device
                yield name, base[name], change, words
    for change, words in ((dict(groups=3), "groups"), (dict(groups=8, top_groups=1), "fewer than"), (dict(logits=torch.zeros(1, 8).expand(1 << 30, 8)), "30 bits"),
                          (dict(logits=torch.zeros(1, 8).expand((1 << 28) + 1, 8), k=8), "30 bits")):
        yield "route", base["route"], change, words


@pytest.mark.parametrize("name, base, change, words", list(refusals()))
def test_tensors_without_data_meet_the_same_checks(name, base, change, words):
    def moved(kw):
        return {n: v.to("meta") if isinstance(v, torch.Tensor) else v for n, v in kw.items()}
    op = getattr(torch.ops.fr_hip, name)
    op(**moved(base))
    with pytest.raises(RuntimeError, match=words):
        op(**moved({**base, **change}))
