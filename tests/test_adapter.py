"""Adapter operators (adapter.py, ops.py, csrc/k_linear, k_norm, k_route): refusals on the CPU, numerics on the GPU.

Tolerances, from arithmetic alone.  u(t) = eps / 2 of a type is the most one rounding is off, relative; U = u(f32).
A sum of n products in f32, in any order, is off by at most n U times the sum of their magnitudes (to first order; 1.01
covers the rest), on top of which every further f32 operation adds one U of its result.  Activations: slope at most 1.13
(GELU; SiLU 1.10, the rest 1), evaluated within 8 U of their result plus 8 U of the argument's error through expf.
"""
import ctypes as C
import math

import pytest
import torch

import face_recognition_amd as fr
from face_recognition_amd import _lib, adapter, ops
from oracle import adapter as oa

U = 2.0 ** -24
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
MOST = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 1e-37, torch.float16: 2.0 ** -25, torch.float32: 1e-37}       # half a subnormal step (f16)


def gen(seed, device="cuda"):
    return torch.Generator(device=device).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=g.device) * scale).to(dtype)


def close(got, want, tol, what=""):
    """Elementwise; NaN and infinities have to be the same."""
    assert got.shape == want.shape, (got.shape, want.shape)
    got = got.double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    off = ((got - want).abs() - tol)[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()), float((got - want).abs()[fine].max()))


def linear_tol(x, w, bias, residual, want, out):
    K = x.shape[-1]
    mag = x.double().abs() @ w.double().abs().T
    if bias is not None:
        mag = mag + bias.double().abs()
    tol = 1.13 * 1.01 * (K + 1) * U * mag + 16 * U * (want.abs() + mag)
    if residual is not None:
        tol = tol + 2 * U * (residual.double().abs() + want.abs())
    return tol + MOST[out] * (want.abs() + tol) + TINY[out]


# ---- on the CPU: what is refused ---------------------------------------------------------------------------------------

def test_module_is_reachable():
    assert fr.adapter is adapter
    for name in ("linear", "block_norm", "route", "expert_linear"):
        assert hasattr(torch.ops.fr_hip, name)


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 8), torch.zeros(4, 8)
    r = adapter.Routing(torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    for call in (lambda: adapter.linear(x, w), lambda: adapter.block_norm(x), lambda: adapter.route(x, 2),
                 lambda: adapter.expert_linear(x, w[None], r), lambda: adapter.ResidualAdapter(8, 16)(x)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(NotImplementedError):
        torch.ops.fr_hip.linear(x, w, None, None, None, "none", None)


LINEAR = dict(bias=None, slope=None, residual=None, act="none", out_dtype=None)


@pytest.mark.parametrize("change, words", [
    (dict(x=torch.zeros(2, 7)), "weight"), (dict(weight=torch.zeros(4)), "weight"), (dict(weight=torch.zeros(4, 8).half()), "one type"),
    (dict(x=torch.zeros(2, 8, dtype=torch.float64), weight=torch.zeros(4, 8, dtype=torch.float64)), "float32, bfloat16"),
    (dict(bias=torch.zeros(5)), "bias"), (dict(bias=torch.zeros(4).half()), "bias"), (dict(residual=torch.zeros(2, 5)), "residual"),
    (dict(residual=torch.zeros(2, 4, dtype=torch.int32)), "residual"), (dict(act="tanh"), "act"), (dict(act="prelu"), "slope"),
    (dict(slope=torch.zeros(4)), "slope"), (dict(act="prelu", slope=torch.zeros(4).half()), "slope"), (dict(out_dtype=torch.int8), "out_dtype"),
    (dict(weight=torch.zeros(0, 8)), "weight"), (dict(x=torch.zeros(2, 0), weight=torch.zeros(4, 0)), "weight"),
    (dict(x=torch.zeros(2, 8, requires_grad=True)), "inference only"), (dict(bias=torch.zeros(4, requires_grad=True)), "inference only"),
    (dict(weight=torch.zeros(4, 8, device="meta")), "all tensors on"),
    (dict(x=torch.zeros(1, 1).expand(1, (1 << 32) + 8), weight=torch.zeros(1, 1).expand(4, (1 << 32) + 8)), "31 bits"),
])
def test_linear_refuses(change, words):
    with pytest.raises(RuntimeError, match=words):
        ops._linear(**{**dict(x=torch.zeros(2, 8), weight=torch.zeros(4, 8), **LINEAR), **change})


NORM = dict(residual=None, slot_weights=None, norm="rms", weight=None, bias=None, eps=1e-6, gate=None, gate_act="none", scale=1.0,
            next_norm="none", next_weight=None, next_bias=None, next_eps=1e-6, out_dtype=None, next_dtype=None)


@pytest.mark.parametrize("change, words", [
    (dict(x=torch.tensor(1.0)), "expected x"), (dict(x=torch.zeros(2, 0)), "expected x"), (dict(norm="batch"), "norm"), (dict(next_norm="x"), "next_norm"),
    (dict(norm="l2", weight=torch.ones(8)), "belong"), (dict(norm="none", bias=torch.ones(8)), "belong"),
    (dict(next_weight=torch.ones(8)), "belong"), (dict(weight=torch.ones(7)), "weight"), (dict(weight=torch.ones(8).half()), "weight"),
    (dict(residual=torch.zeros(3, 8)), "residual"), (dict(gate=torch.zeros(2)), "gate"), (dict(gate=torch.zeros(8), gate_act="relu"), "gate_act"),
    (dict(gate=torch.zeros(8, dtype=torch.int64)), "gate"), (dict(slot_weights=torch.zeros(3)), "slot_weights"),
    (dict(slot_weights=torch.zeros(2).half()), "slot_weights"), (dict(x=torch.zeros(2, 8, requires_grad=True)), "inference only"),
    (dict(x=torch.zeros(1, 16385)), "16384"), (dict(x=torch.zeros(1, dtype=torch.float32).expand((1 << 32) + 8)), "16384"),
    (dict(x=torch.zeros(2, 8, dtype=torch.float64)), "float32, bfloat16"), (dict(next_dtype=torch.int32, next_norm="l2"), "next_dtype"),
])
def test_block_norm_refuses(change, words):
    with pytest.raises(RuntimeError, match=words):
        ops._block_norm(**{**dict(x=torch.zeros(2, 8), **NORM), **change})


ROUTE = dict(k=2, score="softmax", bias=None, groups=1, top_groups=1, renormalise=True, scale=1.0)


@pytest.mark.parametrize("change, words", [
    (dict(groups=0), "groups"), (dict(groups=(1 << 32) + 1), "groups"), (dict(groups=2, top_groups=3), "groups"), (dict(groups=4, top_groups=0), "groups"),
    (dict(logits=torch.zeros(8)), "expected logits"), (dict(logits=torch.zeros(2, 0)), "expected logits"), (dict(k=0), "experts"), (dict(k=9), "experts"),
    (dict(score="relu"), "score"), (dict(bias=torch.zeros(7)), "bias"), (dict(bias=torch.zeros(8).half()), "bias"),
    (dict(logits=torch.zeros(2, 8, dtype=torch.int32)), "logits"), (dict(logits=torch.zeros(2, 600)), "512"),
    (dict(logits=torch.zeros(2, 32), k=17), "16"), (dict(logits=torch.zeros(2, 8, requires_grad=True)), "inference only"),
])
def test_route_refuses(change, words):
    with pytest.raises(RuntimeError, match=words):
        ops._route(**{**dict(logits=torch.zeros(2, 8), **ROUTE), **change})


EXPERT = dict(order=torch.zeros(4, dtype=torch.int32), offsets=torch.zeros(4, dtype=torch.int32), k=2, bias=None, act="none", slope=None,
              rows="tokens", out="sorted", out_dtype=None)


@pytest.mark.parametrize("change, words", [
    (dict(x=torch.zeros(2, 7)), "weight"), (dict(weight=torch.zeros(4, 8)), "weight"), (dict(rows="x"), "rows"), (dict(out="x"), "out"),
    (dict(order=torch.zeros(4)), "order"), (dict(order=torch.zeros(4, dtype=torch.int64)), "order"), (dict(offsets=torch.zeros(3, dtype=torch.int32)), "offsets"),
    (dict(k=3), "multiple"), (dict(k=0), "multiple"), (dict(rows="sorted"), "rows of x"), (dict(x=torch.zeros(4, 8)), "rows of x"),
    (dict(bias=torch.zeros(4)), "bias"), (dict(act="prelu"), "slope"), (dict(act="prelu", slope=torch.zeros(4)), "slope"), (dict(act="x"), "act"),
    (dict(weight=torch.zeros(3, 4, 8).half()), "one type"), (dict(out_dtype=torch.float64), "out_dtype"),
    (dict(weight=torch.zeros(3, 4, 8, requires_grad=True)), "inference only"),
])
def test_expert_linear_refuses(change, words):
    with pytest.raises(RuntimeError, match=words):
        ops._expert_linear(**{**dict(x=torch.zeros(2, 8), weight=torch.zeros(3, 4, 8), **EXPERT), **change})


def test_c_entries_refuse_before_they_launch():
    """Every refusal is an fr_status with a message, given before the GPU is touched (there is none here)."""
    lib, one = _lib.lib(), 4096                                # an address that nothing may follow

    def refused(rc, status, words):
        assert rc == status and words in lib.fr_last_error().decode(), (rc, lib.fr_last_error())

    def linear(M=1, N=4, K=8, ldx=8, kind=1, bt=1, rt=1, ot=1, act=0, x=one, slope=None, bias=None, residual=None):
        return lib.fr_linear(x, ldx, one, bias, slope, residual, 4, one, M, N, K, kind, bt, rt, ot, act, None, 0, None)
    refused(linear(M=-1), -1, "shape")
    refused(linear(N=0), -1, "shape")
    refused(linear(K=-8), -1, "shape")
    refused(linear(kind=3), -1, "type")
    refused(linear(bias=one, bt=2), -1, "type")
    refused(linear(residual=one, rt=9), -1, "type")
    refused(linear(act=7), -1, "activation")
    refused(linear(act=1), -1, "slopes")
    refused(linear(x=None), -1, "NULL")
    assert linear(M=0) == 0
    need = C.c_size_t()
    refused(lib.fr_linear_workspace_bytes(1, 0, 1, 0, C.byref(need)), -1, "shape")

    def norm(T=1, d=8, slots=0, kind=1, weight=None, gate=None, ldc=1, ga=0, out=one, nn=0, nout=None, nw=None, x=one):
        return lib.fr_block_norm(x, 1, slots, None, T, d, kind, weight, None, 1e-6, gate, 1, 0, ldc, ga, 1.0, None, 0, out, 1, nn, nw, None, 1e-6, nout, 1, None)
    refused(norm(d=16385), -1, "16384")
    refused(norm(T=-1), -1, "shape")
    refused(norm(slots=2), -1, "slot_weights")
    refused(norm(kind=4), -1, "norm")
    refused(norm(kind=3, weight=one), -1, "belong")
    refused(norm(nw=one), -1, "belong")
    refused(norm(gate=one, ldc=2), -1, "strides")
    refused(norm(gate=one, ga=3), -1, "gate")
    refused(norm(nn=1), -1, "together")
    refused(norm(out=None), -1, "no output")
    refused(norm(x=None), -1, "NULL")
    assert norm(T=0) == 0

    def route(T=1, E=8, k=2, kind=0, score=0, groups=1, top=1, ws=one, wsb=1 << 20):
        return lib.fr_route(one, kind, T, E, k, score, None, groups, top, 1, 1.0, one, one, one, one, ws, wsb, None)
    refused(route(E=513), -1, "512")
    refused(route(E=64, k=17), -1, "16")
    refused(route(k=9), -1, "shape")
    refused(route(T=-1), -1, "shape")
    refused(route(T=1 << 31), -2, "31 bits")
    refused(route(kind=5), -1, "type")
    refused(route(score=2), -1, "score")
    refused(route(groups=3), -1, "groups")
    refused(route(groups=4, top=5), -1, "groups")
    refused(route(groups=8, top=1), -1, "fewer than k")
    refused(route(T=1000, wsb=8), -4, "workspace")
    refused(route(T=1000, ws=None), -4, "workspace")

    def expert(T=1, k=2, E=4, N=8, K=8, kind=1, act=0, order=one):
        return lib.fr_expert_linear(one, 0, one, None, None, order, one, one, 0, T, k, E, N, K, kind, kind, kind, act, None)
    refused(expert(E=0), -1, "shape")
    refused(expert(k=0), -1, "shape")
    refused(expert(T=1 << 30, k=2), -2, "31 bits")
    refused(expert(kind=4), -1, "type")
    refused(expert(act=8), -1, "activation")
    refused(expert(act=1), -1, "slopes")
    refused(expert(order=None), -1, "NULL")
    assert expert(T=0) == 0


@pytest.mark.parametrize("M, K", [(1, 1), (1, 8), (64, 1), (65, 8), (1, 512)])
def test_c_entries_refuse_outputs_wider_than_a_launch(M, K):
    """N of nearly 31 bits: the tiles are counted in 64 bits and refused before anything is launched."""
    lib, at, need = _lib.lib(), 4096, C.c_size_t()
    for N in (2 ** 31 - 1, 2 ** 31 - 8, 2 ** 31 - 64):
        assert lib.fr_linear_workspace_bytes(M, N, K, _lib.FR_TYPE_BF16, C.byref(need)) == 0
        assert need.value == 0
        rc = lib.fr_linear(at, K, at, None, None, None, 0, at, M, N, K, 1, 1, 1, 1, 0, None, 0, None)
        assert rc != 0 and b"tiles" in lib.fr_last_error()
        rc = lib.fr_expert_linear(at, 0, at, None, None, at, at, at, 0, M, 1, 1, N, K, 1, 1, 1, 0, None)
        assert rc != 0 and b"tiles" in lib.fr_last_error()


@pytest.mark.gpu
def test_plans_refuse_the_new_activations():
    w = torch.zeros(8, 8, 1, 1)
    for code in (_lib.FR_ACT_GELU, _lib.FR_ACT_SILU):
        d = (_lib.LayerDesc * 1)()
        d[0].op, d[0].src, d[0].residual, d[0].cin, d[0].cout = _lib.FR_OP_CONV, -1, -1, 8, 8
        d[0].kernel, d[0].stride, d[0].pad, d[0].groups, d[0].act, d[0].weight = 1, 1, 0, 1, code, w.data_ptr()
        h = C.c_void_p()
        assert _lib.lib().fr_plan_create(d, 1, 8, 4, 4, _lib.FR_PREC_BF16, C.byref(h)) == -2


def test_blocks_refuse():
    for bad in (dict(norm="l2"), dict(act="prelu"), dict(act="x"), dict(dtype=torch.float64)):
        with pytest.raises(ValueError):
            adapter.ResidualAdapter(8, 16, **bad)
    block = adapter.ExpertAdapter(8, 16, experts=4)
    assert not any(p.requires_grad for p in block.parameters())
    again = adapter.ExpertAdapter(8, 16, experts=4)
    again.load_state_dict(block.state_dict())


def test_shapes_without_data():
    """Meta tensors take the same checks."""
    x, w = torch.empty(3, 5, 8, device="meta"), torch.empty(6, 8, device="meta")
    assert torch.ops.fr_hip.linear(x, w, None, None, None, "none", torch.float32).shape == (3, 5, 6)
    out, nxt = torch.ops.fr_hip.block_norm(x, None, torch.empty(3, 5, device="meta"), "rms", None, None, 1e-6, None, "none", 1.0, "l2", None, None, 1e-6,
                                           None, torch.bfloat16)
    assert out.shape == nxt.shape == (3, 8) and nxt.dtype == torch.bfloat16
    assert [t.shape for t in torch.ops.fr_hip.route(w, 2, "softmax", None, 1, 1, True, 1.0)] == [(6, 2), (6, 2), (12,), (9,)]
    with pytest.raises(RuntimeError):
        torch.ops.fr_hip.linear(x, w.t(), None, None, None, "none", None)


# ---- on the GPU: linear ------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m, k, n", [(1, 512, 2048), (1, 1, 1), (2, 7, 3), (5, 129, 65), (16, 64, 16), (17, 4096, 200), (33, 100, 130),
                                     (64, 512, 512), (65, 72, 64), (128, 128, 256), (130, 264, 257), (300, 513, 130), (513, 2048, 96), (257, 520, 1032)])
def test_linear_shapes(kind, m, k, n):
    g, dt = gen(m * 7 + k * 3 + n), TYPES[kind]
    x, w, b = randn(g, m, k, dtype=dt), randn(g, n, k, dtype=dt, scale=k ** -0.5), randn(g, n, dtype=dt)
    want = oa.linear(x, w, b)
    got = adapter.linear(x, w, b)
    assert got.dtype == dt
    close(got, want, linear_tol(x, w, b, None, want, dt), (kind, m, k, n))


@pytest.mark.gpu
@pytest.mark.parametrize("kind, out, res", [("bf16", "bf16", "bf16"), ("bf16", "f32", "f32"), ("f16", "f16", "f32"), ("f32", "bf16", "f16"), ("f32", "f32", "f32")])
@pytest.mark.parametrize("act", ["none", "prelu", "hswish", "relu", "hsigmoid", "gelu", "silu"])
@pytest.mark.parametrize("m, k, n", [(3, 96, 70), (200, 96, 136), (700, 160, 520)])
def test_linear_epilogues(kind, out, res, act, m, k, n):
    g, dt = gen(11), TYPES[kind]
    x, w = randn(g, m, k, dtype=dt, scale=3), randn(g, n, k, dtype=dt, scale=k ** -0.5)
    b, r = randn(g, n), randn(g, m, n, dtype=TYPES[res])
    slope = randn(g, n) if act == "prelu" else None
    want = oa.linear(x, w, b, slope, r, act)
    got = adapter.linear(x, w, b, act=act, slope=slope, residual=r, out_dtype=TYPES[out])
    assert got.dtype == TYPES[out]
    tol = linear_tol(x, w, b, r, want, TYPES[out])
    if act == "prelu":
        tol = tol * slope.abs().clamp_min(1.0).double()
    close(got, want, tol, (kind, out, act))


@pytest.mark.gpu
def test_linear_strides_and_dims():
    g = gen(5)
    wide, w = randn(g, 40, 300, dtype=torch.bfloat16), randn(g, 24, 128, dtype=torch.bfloat16)
    for x in (wide[:, :128], wide[:, 3:131], wide[::2, 8:136], wide[:1, :128].expand(40, 128), wide.t()[:128, :].t(), wide[:, :128].reshape(4, 10, 128),
              wide[0, :128], wide[:0, :128]):
        want = oa.linear(x, w)
        got = adapter.linear(x, w)
        assert got.shape == x.shape[:-1] + (24,)
        close(got, want, linear_tol(x, w, None, None, want, torch.bfloat16))
    res = randn(g, 40, 50, dtype=torch.bfloat16)[:, 5:29]
    x = wide[:, :128]
    want = oa.linear(x, w, residual=res)
    close(adapter.linear(x, w, residual=res), want, linear_tol(x, w, None, res, want, torch.bfloat16))
    wt = randn(g, 128, 24, dtype=torch.bfloat16).t()           # weights that lie the other way are laid out within the call
    want = oa.linear(x, wt)
    close(adapter.linear(x, wt), want, linear_tol(x, wt, None, None, want, torch.bfloat16))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m, k, n", [(1, 64, 32), (70, 72, 72), (300, 136, 264)])
def test_linear_keeps_infinities_and_nans_in_their_rows(kind, m, k, n):
    """A row of x that is not finite spoils its own outputs and no other row's; neither do rows behind a matrix's end."""
    g, dt = gen(6), TYPES[kind]
    store = torch.full((m + 200, k), math.nan, device="cuda", dtype=dt)
    store[:m] = randn(g, m, k, dtype=dt)
    x, w = store[:m], randn(g, n, k, dtype=dt)
    x[0, 0] = math.inf
    if m > 1:
        x[m // 2, 3] = math.nan
    want = oa.linear(x, w)
    finite = torch.where(torch.isfinite(x), x, torch.zeros((), dtype=dt, device="cuda"))
    close(adapter.linear(x, w), want, linear_tol(finite, w, None, None, torch.nan_to_num(want, posinf=0, neginf=0), dt))


@pytest.mark.gpu
def test_linear_extremes_of_activations():
    """Large arguments either way: no overflow inside, limits as the functions have them."""
    x = torch.tensor([-1e30, -200.0, -90.0, -40.0, -13.0, -5.5, -1e-20, 0.0, 1e-20, 5.5, 40.0, 200.0, 1e30], device="cuda")[:, None]
    w = torch.ones(1, 1, device="cuda")
    for act in ("hswish", "relu", "hsigmoid", "gelu", "silu"):
        want = oa.act(x, act)
        # exp2(y) is off by U of y's rounding times |y| <= 128 in its exponent (89 U), and that of v^2 by as much again: 200 U
        # covers both.  e^88.73 is the last in f32's range: below that SiLU is 0 where |v| e^v < 88.73 * 2^-128 < 2^-121.
        close(adapter.linear(x, w, act=act), want, 200 * U * want.abs() + 2.0 ** -121, act)
        ends = torch.tensor([math.inf, -math.inf, math.nan], device="cuda")[:, None]
        close(adapter.linear(ends, w, act=act), oa.act(ends, act), torch.zeros((), dtype=torch.float64, device="cuda"), act)


@pytest.mark.gpu
def test_linear_residual_may_be_wide_or_missing_and_rows_beyond_31_bits():
    """x rows whose byte offsets pass 32 bits."""
    rows, k = 70000, 32768                                     # 4.6 GB of bf16
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    g = gen(9)
    x[-3:] = randn(g, 3, k, dtype=torch.bfloat16)
    x[1] = x[-1]
    w = randn(g, 16, k, dtype=torch.bfloat16, scale=k ** -0.5)
    got = adapter.linear(x, w, out_dtype=torch.float32)
    want = oa.linear(x[-3:], w)
    close(got[-3:], want, linear_tol(x[-3:], w, None, None, want, torch.float32))
    assert torch.equal(got[1], got[-1]) and not got[2:-3].any()


@pytest.mark.gpu
def test_linear_same_bits_every_time():
    g = gen(12)
    for m, k, n in ((8, 4096, 1024), (100, 4096, 300), (1000, 1024, 512)):
        x, w = randn(g, m, k, dtype=torch.bfloat16), randn(g, n, k, dtype=torch.bfloat16)
        first = adapter.linear(x, w)
        assert all(torch.equal(first, adapter.linear(x, w)) for _ in range(3))


# ---- on the GPU: block_norm --------------------------------------------------------------------------------------------

def norm_ref(x, residual=None, slot_weights=None, norm="rms", weight=None, bias=None, eps=1e-6, gate=None, gate_act="none", scale=1.0,
             next_norm=None, next_weight=None, next_bias=None, next_eps=1e-6, out_dtype=None, next_dtype=None):
    """(out, next, tolerance of out, of next) with the bounds of one row:
    y: slots U of the sum of magnitudes; the statistics d U relative (of the row's magnitude for the mean); a few U a step."""
    y = x.double() if slot_weights is None else oa.weighted(x, slot_weights)
    mag = y.abs() if slot_weights is None else oa.weighted(x.double().abs(), slot_weights.abs())
    slots = 0 if slot_weights is None else x.shape[-2]
    err = (slots + 1) * U * mag if slots else torch.zeros_like(y)
    d = y.shape[-1]

    def normed(v, e, name, w, b, ep):
        n = oa.norm(v, name, w, b, ep)
        if name == "none":
            return n, e
        c = v - v.mean(-1, keepdim=True) if name == "layer" else v
        if name == "layer":
            e = e + (d + 2) * U * v.abs().mean(-1, keepdim=True) + e.mean(-1, keepdim=True) + U * c.abs()
        s = c.pow(2).mean(-1, keepdim=True) + (ep if name != "l2" else 0)
        inv = torch.where(s > 0, s.rsqrt() if name != "l2" else (s * d).rsqrt(), torch.zeros_like(s))
        # d(1/sqrt(s)) / (1/sqrt(s)) = half of ds / s: the sum's d U, and the elements' own errors
        rel = (d + 8) * U + (c.abs() * e).mean(-1, keepdim=True) / s.clamp_min(1e-300)
        wd = 1.0 if w is None else w.double().abs()
        return n, (e * inv + c.abs() * inv * (rel + 8 * U)) * wd + 2 * U * n.abs()

    v, err = normed(y, err, norm, weight, bias, eps)
    if gate is not None:
        gd = oa.gate_of(gate, gate_act)
        v, err = v * gd, err * gd.abs() + 16 * U * (v * gd).abs()
    v, err = v * scale, err * abs(scale) + U * (v * scale).abs()
    if residual is not None:
        v = v + residual.double()
        err = err + U * v.abs()
    out = out_dtype or x.dtype
    tol = err + MOST[out] * (v.abs() + err) + TINY[out]
    if next_norm is None:
        return v, None, tol, None
    n, e = normed(v, err, next_norm, next_weight, next_bias, next_eps)
    kind = next_dtype or out
    return v, n, tol, e + MOST[kind] * (n.abs() + e) + TINY[kind]


def check_norm(x, *args, what="", **kw):
    got = adapter.block_norm(x, *args, **kw)
    want, nxt, tol, ntol = norm_ref(x, *args, **kw)
    if nxt is None:
        close(got, want, tol, what)
    else:
        close(got[0], want, tol, what)
        close(got[1], nxt, ntol, what)
        assert got[1].dtype == (kw.get("next_dtype") or kw.get("out_dtype") or x.dtype)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("norm", ["none", "rms", "layer", "l2"])
@pytest.mark.parametrize("t, d", [(1, 1), (3, 7), (5, 512), (4, 513), (9, 1000), (2, 1025), (7, 2048), (3, 4099), (2, 8192), (2, 16384), (1, 16381), (300, 64)])
def test_block_norm_shapes(kind, norm, t, d):
    g, dt = gen(t + d), TYPES[kind]
    x = randn(g, t, d, dtype=dt, scale=2) + 0.5
    w = 1 + randn(g, d, scale=0.2) if norm in ("rms", "layer") else None
    b = randn(g, d) if norm == "layer" else None
    check_norm(x, norm=norm, weight=w, bias=b, what=(kind, norm, t, d))


@pytest.mark.gpu
@pytest.mark.parametrize("gate, gate_act", [("none", "none"), ("channel", "sigmoid"), ("row", "tanh"), ("full", "none")])
@pytest.mark.parametrize("slots", [0, 1, 2, 5])
@pytest.mark.parametrize("next_norm", [None, "rms", "layer", "l2"])
@pytest.mark.parametrize("d", [200, 512, 1111, 3000])
def test_block_norm_fused(gate, gate_act, slots, next_norm, d):
    g, t = gen(d + slots), 11
    x = randn(g, t, slots, d, dtype=torch.bfloat16) if slots else randn(g, t, d, dtype=torch.bfloat16)
    sw = torch.rand(t, slots, generator=g, device="cuda") if slots else None
    shape = {"none": None, "channel": (d,), "row": (t, 1), "full": (t, d)}[gate]
    kw = dict(slot_weights=sw, norm="layer" if d == 512 else "rms", weight=1 + randn(g, d, scale=0.1), gate=randn(g, *shape, dtype=torch.float16) if shape else None,
              gate_act=gate_act, scale=0.7, out_dtype=torch.float32)
    if next_norm:
        kw.update(next_norm=next_norm, next_dtype=torch.bfloat16)
        if next_norm != "l2":
            kw.update(next_weight=1 + randn(g, d, scale=0.1))
        if next_norm == "layer":
            kw.update(next_bias=randn(g, d))
    check_norm(x, randn(g, t, d), what=(gate, slots, next_norm, d), **kw)


@pytest.mark.gpu
def test_block_norm_rows_that_say_nothing():
    """Zero rows, slots of weight 0 that hold NaN, rows without any slot, padded shapes, no rows."""
    g = gen(3)
    x = randn(g, 4, 3, 512, dtype=torch.bfloat16)
    sw = torch.rand(4, 3, generator=g, device="cuda")
    x[1, 2], sw[1, 2] = math.nan, 0.0
    x[2], sw[2] = math.inf, 0.0
    res = randn(g, 4, 512)
    out, rows = check_norm(x, res, slot_weights=sw, next_norm="l2", out_dtype=torch.float32, next_dtype=torch.bfloat16)
    assert torch.equal(out[2], res[2])
    zero = torch.zeros(3, 100, device="cuda")
    for norm in ("none", "rms", "layer", "l2"):
        assert not adapter.block_norm(zero, norm=norm).any()
    assert adapter.block_norm(zero[:0]).shape == (0, 100)
    out, nxt = adapter.block_norm(zero[:0], next_norm="l2")
    assert out.shape == nxt.shape == (0, 100)
    assert adapter.block_norm(randn(g, 2, 3, 64)).shape == (2, 3, 64)


@pytest.mark.gpu
def test_block_norm_keeps_nan_in_its_row():
    g = gen(4)
    x = randn(g, 6, 512)
    x[2, 100] = math.nan
    x[4, 7] = math.inf
    got = adapter.block_norm(x, norm="layer")
    alone = [adapter.block_norm(x[i:i + 1], norm="layer")[0] for i in (0, 1, 3, 5)]
    assert torch.isnan(got[2]).all() and torch.isnan(got[4]).all()
    assert torch.equal(got[[0, 1, 3, 5]], torch.stack(alone))


@pytest.mark.gpu
def test_block_norm_strides_and_alignment():
    g = gen(8)
    store = randn(g, 20, 1030, dtype=torch.bfloat16)
    check_norm(store[:, 3:515], store[:, 515:1027], norm="rms")
    check_norm(store.view(-1)[1:1 + 512 * 7].view(7, 512), norm="layer", gate=store.view(-1)[3:515])
    check_norm(store[:1].expand(5, 1030), norm="rms", weight=randn(g, 1031)[1:])
    check_norm(store.t().contiguous().t(), norm="l2")


@pytest.mark.gpu
def test_block_norm_small_and_large_rows():
    """Embeddings of untrained nets are around 1e-14, raw logits may be huge: unit rows either way."""
    g = gen(10)
    for scale in (1e-14, 1e-9, 1.0, 1e12):
        x = randn(g, 3, 512, scale=scale)
        check_norm(x, norm="l2")
        check_norm(x, norm="rms")
    got = adapter.block_norm(randn(g, 3, 512, scale=1e-14), norm="none", next_norm="l2", next_dtype=torch.bfloat16)[1]
    assert ((got.double().norm(dim=1) - 1).abs() < 2.0 ** -8).all()


@pytest.mark.gpu
def test_block_norm_many_rows():
    g = gen(13)
    x = randn(g, 70001, 512, dtype=torch.bfloat16)
    check_norm(x, norm="rms")
    big = torch.zeros(300000, 8192, dtype=torch.bfloat16, device="cuda")        # 4.9 GB: offsets pass 32 bits
    big[-1] = x[:16].reshape(-1)
    big[0] = big[-1]
    got = adapter.block_norm(big, norm="rms")
    assert torch.equal(got[0], got[-1]) and not got[1:-1].any()
    check_norm(big[-1:], norm="rms")


@pytest.mark.gpu
@pytest.mark.parametrize("d", [8, 2056])
def test_block_norm_more_rows_than_a_launch(d):
    """2^22 rows a launch."""
    t = 4200001 if d == 8 else 4194307
    x = randn(gen(14), t, d, dtype=torch.bfloat16)
    got = adapter.block_norm(x, norm="layer")
    for at in (0, 4194296, t - 8):
        if at < t:
            part = x[at:at + 8]
            want, _, tol, _ = norm_ref(part, norm="layer")
            close(got[at:at + 8], want, tol, at)
    # rows of every block and turn, against the same rows in a small call
    pick = torch.randint(0, t, (5000,), generator=gen(15), device="cuda")
    assert torch.equal(got[pick], adapter.block_norm(x[pick], norm="layer"))


# ---- on the GPU: route -------------------------------------------------------------------------------------------------

def check_route(logits, k, what="", **kw):
    got = adapter.route(logits, k, **kw)
    w, e, order, offsets = oa.route(logits, k, **kw)
    assert torch.equal(got.experts.cpu(), e), what
    assert torch.equal(got.order.cpu(), order), what
    assert torch.equal(got.offsets.cpu(), offsets), what
    # expf: its argument is a difference of logits rounded once (U of it through the exponential: at most 104 U before the
    # result is below f32's range), a sum of up to E of them, a division and a scale
    tol = (128 + logits.shape[1]) * U * w.abs() + 2.0 ** -126
    close(got.weights.cpu(), w, tol, what)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("t, e, k, groups, top", [(1, 1, 1, 1, 1), (1, 64, 4, 1, 1), (3, 5, 5, 1, 1), (65, 65, 3, 1, 1), (130, 8, 2, 4, 2), (77, 256, 8, 8, 4),
                                                  (40, 512, 16, 64, 9), (33, 100, 7, 10, 3), (200, 16, 1, 16, 5), (10, 384, 8, 2, 1), (1000, 32, 4, 1, 1)])
def test_route_shapes(kind, score, biased, t, e, k, groups, top):
    g = gen(t + e + k)
    logits = randn(g, t, e, dtype=TYPES[kind], scale=1.5)
    bias = randn(g, e, scale=0.2) if biased else None
    check_route(logits, k, score=score, bias=bias, groups=groups, top_groups=top, what=(kind, score, biased, t, e, k, groups))


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalise, scale", [(False, 1.0), (True, 2.5), (False, 0.5)])
def test_route_weights(score, renormalise, scale):
    g = gen(21)
    check_route(randn(g, 50, 24, scale=4), 5, score=score, renormalise=renormalise, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups, top", [(1, 1), (4, 2)])
def test_route_ties_go_to_the_lower_index(score, groups, top):
    g = gen(22)
    logits = torch.randint(0, 3, (100, 32), generator=g, device="cuda").float()
    check_route(logits, 6, score=score, groups=groups, top_groups=top)
    check_route(torch.zeros(70, 32, device="cuda"), 6, score=score, groups=groups, top_groups=top)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups, top, biased", [(1, 1, False), (1, 1, True), (4, 2, True)])
def test_route_masks(score, groups, top, biased):
    """-inf and NaN mask; rows with fewer experts than k, and with none."""
    g = gen(23)
    logits = randn(g, 90, 32)
    logits[torch.rand(90, 32, generator=g, device="cuda") < 0.6] = -math.inf
    logits[0], logits[40:45], logits[-1] = -math.inf, -math.inf, math.nan
    logits[3, 5], logits[4, 6], logits[5, 1:] = math.nan, math.inf, -math.inf
    bias = randn(g, 32, scale=0.1) if biased else None
    if biased:
        bias[7] = -math.inf
    got = check_route(logits, 4, score=score, bias=bias, groups=groups, top_groups=top)
    assert (got.experts[40:45] == -1).all() and not got.weights[40:45].any()


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_route_extreme_logits(score):
    """Logits as far apart as f32 goes, all very low (sigmoids below f32's range), the type's lowest value."""
    g = gen(24)
    for scale, shift in ((1.0, -150.0), (30.0, 0.0), (1.0, 1e4), (1e30, 0.0)):
        check_route(randn(g, 40, 16, scale=scale) + shift, 3, score=score, what=(scale, shift))
    low = torch.full((4, 16), torch.finfo(torch.float32).min, device="cuda")
    low[1, 3] = 0.0
    check_route(low, 3, score=score)


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [1, 2])
def test_route_scores_closer_than_a_float_step(groups):
    """Biased sigmoids whose exact order a float cannot see."""
    E = 32
    l = torch.full((64, E), 3.0, device="cuda")
    l += torch.arange(E, device="cuda") * 2.0 ** -21 * torch.where(torch.arange(64, device="cuda") % 2 == 0, 1.0, -1.0)[:, None]
    check_route(l, 5, score="sigmoid", bias=torch.full((E,), 0.25, device="cuda"), groups=groups, top_groups=1)
    check_route(l, 5, score="softmax", bias=torch.full((E,), 100.0, device="cuda"), groups=groups, top_groups=1)


@pytest.mark.gpu
def test_route_many_rows():
    """Against torch in 64 bits: sizes the row by row oracle is too slow for; every chunk's and block's borders."""
    for t, e, k in ((65536 + 3, 64, 4), (20001, 256, 8), (4096, 512, 16)):
        g = gen(t)
        logits = randn(g, t, e)
        got = adapter.route(logits, k)
        best = torch.sort(logits, dim=-1, descending=True, stable=True)
        assert torch.equal(got.experts.long(), best.indices[:, :k])
        want = torch.softmax(best.values[:, :k].double(), -1)
        close(got.weights, want, 256 * U * want)
        flat = torch.sort(best.indices[:, :k].reshape(-1), stable=True)
        assert torch.equal(got.order.long(), flat.indices)
        assert torch.equal(got.offsets.long(), torch.searchsorted(flat.values, torch.arange(e + 1, device="cuda")))


@pytest.mark.gpu
@pytest.mark.parametrize("e, k", [(8, 2), (64, 4), (100, 3), (256, 8), (500, 10)])
@pytest.mark.parametrize("t", [2, 4, 5, 9, 31, 32, 33, 63, 64, 65, 129])
def test_route_few_rows(e, k, t):
    g = gen(t + e)
    check_route(randn(g, t, e), k, (t, e, k))
    check_route(randn(g, t, e, dtype=torch.bfloat16), k, (t, e, k), score="sigmoid", bias=randn(g, e, scale=0.1))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("e, k, groups, top", [(204, 8, 4, 4), (16, 4, 2, 1), (64, 6, 8, 3), (500, 10, 20, 7), (480, 5, 32, 32)])
def test_route_equal_logits_in_groups(kind, score, e, k, groups, top):
    """16-bit logits without a bias: many equal ones; ones that differ and have the same score in doubles; masks."""
    g, kw = gen(e + k), dict(score=score, groups=groups, top_groups=top)
    x = randn(g, 70, e, dtype=TYPES[kind])
    for what, l in (("random", x), ("few values", (x.float() * 2).round().to(x.dtype) / 2), ("near 1", x + 25), ("at 1", x * 4 + 60), ("low", x * 30 - 590),
                    ("tiny", x * 1e-7 if kind == "f16" else x * 1e-30), ("some tiny", torch.where(x > 0.5, x * (1e-6 if kind == "f16" else 1e-20), x.abs() * -3)),
                    ("zeros", torch.where(x > 0, 0.0, -0.0).to(x.dtype)), ("wide", x * 300), ("masked", x.masked_fill(randn(g, 70, e) > 0.3, -math.inf))):
        check_route(l, k, what=(kind, score, e, what), **kw)


@pytest.mark.gpu
def test_route_nothing():
    got = adapter.route(torch.zeros(0, 12, device="cuda"), 3)
    assert got.weights.shape == got.experts.shape == (0, 3) and got.order.shape == (0,) and got.offsets.tolist() == [0] * 13


# ---- on the GPU: expert_linear -----------------------------------------------------------------------------------------

def choose(g, t, e, k, lost=0.0):
    ex = torch.stack([torch.randperm(e, generator=g, device="cuda")[:k] for _ in range(t)]).to(torch.int32) if t else torch.zeros(0, k, dtype=torch.int32, device="cuda")
    if lost:
        ex[torch.rand(t, k, generator=g, device="cuda") < lost] = -1
    order, offsets = oa.routing_of(ex, e)
    return adapter.Routing((ex >= 0).float() / k, ex, order, offsets)


def check_expert(x, w, r, bias=None, slope=None, act="none", rows="tokens", out="sorted", out_dtype=None, what=""):
    got = adapter.expert_linear(x, w, r, bias, act=act, slope=slope, rows=rows, out=out, out_dtype=out_dtype)
    want = oa.expert_linear(x, w, r.experts, bias, slope, act, rows == "tokens", out == "slots")
    mag = oa.expert_linear(x.double().abs(), w.double().abs(), r.experts, None if bias is None else bias.abs(), None, "none", rows == "tokens", out == "slots")
    kind = out_dtype or x.dtype
    tol = 1.13 * 1.01 * (x.shape[1] + 1) * U * mag + 16 * U * (want.abs() + mag)
    if slope is not None:
        tol = tol * max(1.0, float(slope.abs().max()))
    close(got, want, tol + MOST[kind] * (want.abs() + tol) + TINY[kind], what)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows, out", [("tokens", "sorted"), ("sorted", "slots"), ("tokens", "slots"), ("sorted", "sorted")])
@pytest.mark.parametrize("t, e, k, d, n", [(1, 4, 1, 64, 32), (1, 8, 2, 512, 96), (5, 32, 2, 96, 130), (37, 3, 2, 100, 70), (130, 5, 3, 72, 65), (257, 2, 1, 264, 136),
                                           (90, 70, 4, 33, 17), (600, 2, 2, 128, 264)])
def test_expert_linear_shapes(kind, rows, out, t, e, k, d, n):
    g, dt = gen(t + e + d), TYPES[kind]
    r = choose(g, t, e, k)
    x = randn(g, t if rows == "tokens" else t * k, d, dtype=dt)
    w, b = randn(g, e, n, d, dtype=dt, scale=d ** -0.5), randn(g, e, n, dtype=dt)
    check_expert(x, w, r, b, rows=rows, out=out, what=(kind, rows, out, t, e, k, d, n))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "prelu", "hswish", "relu", "hsigmoid", "gelu", "silu"])
@pytest.mark.parametrize("out", ["sorted", "slots"])
def test_expert_linear_epilogues(act, out):
    g = gen(31)
    r = choose(g, 60, 4, 2)
    x, w, b = randn(g, 60, 64, dtype=torch.bfloat16, scale=3), randn(g, 4, 48, 64, dtype=torch.bfloat16, scale=0.2), randn(g, 4, 48)
    check_expert(x, w, r, b, randn(g, 4, 48) if act == "prelu" else None, act, out=out, out_dtype=torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("out", ["sorted", "slots"])
@pytest.mark.parametrize("t", [3, 200])
def test_expert_linear_slots_without_an_expert(out, t):
    """They get zeros, whatever their rows hold, and what lay in the output's memory does not show."""
    g = gen(32)
    for lost in (0.5, 1.0):
        r = choose(g, t, 6, 3, lost)
        x = randn(g, t, 64, dtype=torch.bfloat16)
        x[(r.experts < 0).all(1)] = math.nan
        w = randn(g, 6, 200, 64, dtype=torch.bfloat16)
        torch.full((t * 3, 200), math.nan, dtype=torch.bfloat16, device="cuda")
        check_expert(x, w, r, out=out)


@pytest.mark.gpu
def test_expert_linear_lopsided():
    """All rows to one expert; experts without a row, first, last and between."""
    g = gen(33)
    x, w = randn(g, 700, 96, dtype=torch.bfloat16), randn(g, 9, 72, 96, dtype=torch.bfloat16)
    for e in (0, 4, 8):
        ex = torch.full((700, 1), e, dtype=torch.int32, device="cuda")
        order, offsets = oa.routing_of(ex, 9)
        check_expert(x, w, adapter.Routing(torch.ones(700, 1, device="cuda"), ex, order, offsets))


@pytest.mark.gpu
def test_expert_linear_tables_that_lie_are_not_followed():
    """Order entries and offsets outside the slots: nothing outside the tensors is read or written, good slots stay right."""
    g = gen(34)
    r = choose(g, 40, 4, 2)
    x, w = randn(g, 40, 64, dtype=torch.bfloat16), randn(g, 4, 32, 64, dtype=torch.bfloat16)
    want = adapter.expert_linear(x, w, r, out="slots")
    order = r.order.clone()
    spoilt = order[5].item(), order[60].item()
    order[5], order[60] = 1 << 30, -7
    got = adapter.expert_linear(x, w, r._replace(order=order), out="slots")
    keep = torch.ones(80, dtype=torch.bool)
    keep[list(spoilt)] = False
    assert torch.equal(got.view(80, 32)[keep.cuda()], want.view(80, 32)[keep.cuda()])
    offsets = r.offsets.clone()
    offsets[-1] = 1 << 30
    adapter.expert_linear(x, w, r._replace(offsets=offsets), out="slots")
    adapter.expert_linear(x, w, r._replace(offsets=-offsets), out="sorted")
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ["tokens", "sorted"])
def test_expert_linear_rows_beyond_32_bits(rows):
    """x of more than 4 GiB, gathered and in the order's positions."""
    t, e, k, d, n = 2200000, 3, 1, 1024, 40                    # 4.5 GB of bf16
    g = gen(35)
    x = torch.zeros(t, d, dtype=torch.bfloat16, device="cuda")
    some = torch.tensor([0, 1, 1000000, t - 2, t - 1], device="cuda")
    x[some] = randn(g, 5, d, dtype=torch.bfloat16)
    ex = (torch.arange(t, device="cuda") % e).to(torch.int32)[:, None]
    flat = torch.sort(ex.reshape(-1), stable=True)
    r = adapter.Routing(torch.ones(t, 1, device="cuda"), ex, flat.indices.to(torch.int32),
                        torch.searchsorted(flat.values, torch.arange(e + 1, device="cuda", dtype=torch.int32)).to(torch.int32))
    w = randn(g, e, n, d, dtype=torch.bfloat16, scale=d ** -0.5)
    got = adapter.expert_linear(x, w, r, rows=rows, out="slots" if rows == "tokens" else "sorted", out_dtype=torch.float32).view(t, n)
    for i in some.tolist():
        slot = i if rows == "tokens" else int(r.order[i])      # sorted: row i stands at position i of the order
        m = w[int(ex[slot])]
        want = oa.linear(x[i][None], m)
        close(got[i][None], want, linear_tol(x[i][None], m, None, None, want, torch.float32), (rows, i))
    keep = torch.ones(t, dtype=torch.bool, device="cuda")
    keep[some] = False
    assert not got[keep].any()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m, k, n", [(1100, 333, 1100), (1300, 130, 1500), (2000, 65, 2000), (1500, 519, 1030)])
def test_linear_large_rows_of_any_alignment(kind, m, k, n):
    g, dt = gen(m + k), TYPES[kind]
    x, w, b = randn(g, m, k, dtype=dt), randn(g, n, k, dtype=dt, scale=k ** -0.5), randn(g, n)
    want = oa.linear(x, w, b, name="relu")
    close(adapter.linear(x, w, b, act="relu"), want, linear_tol(x, w, b, None, want, dt), (kind, m, k, n))
    shifted = torch.empty(m * 384 + 8, dtype=dt, device="cuda")[3:3 + m * 384].view(m, 384)      # whole chunks a row, but not at 16 bytes
    shifted.copy_(randn(g, m, 384, dtype=dt))
    w = randn(g, n, 384, dtype=dt, scale=0.05)
    want = oa.linear(shifted, w)
    close(adapter.linear(shifted, w), want, linear_tol(shifted, w, None, None, want, dt), "shifted")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m, k, n", [(2000, 1032, 1999), (1900, 520, 1700), (2047, 2056, 1030), (4622, 328, 2599), (5865, 136, 2633), (5014, 72, 1409),
                                     (5821, 168, 131), (300, 648, 1500), (5726, 8, 140), (2048, 1024, 2048), (8866, 424, 69), (8831, 168, 1732)])
def test_linear_every_tile(kind, m, k, n):
    """Sizes at which each of the tiles is the estimated best, in one type or the other."""
    g, dt = gen(m + k), TYPES[kind]
    x, w, b, res = randn(g, m, k, dtype=dt), randn(g, n, k, dtype=dt, scale=k ** -0.5), randn(g, n), randn(g, m, n, dtype=dt)
    want = oa.linear(x, w, b, residual=res, name="relu")
    close(adapter.linear(x, w, b, residual=res, act="relu"), want, linear_tol(x, w, b, res, want, dt), (kind, m, k, n))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("m, k, n", [(156, 3937, 200), (65, 1025, 70), (300, 2051, 129), (90, 1333, 1000)])
def test_linear_odd_rows_in_parts(kind, m, k, n):
    """Rows of any alignment whose K is split over parts."""
    g, dt = gen(m + k), TYPES[kind]
    x, w, b, res = randn(g, m, k, dtype=dt), randn(g, n, k, dtype=dt, scale=k ** -0.5), randn(g, n), randn(g, m, n, dtype=dt)
    want = oa.linear(x, w, b, residual=res, name="silu")
    close(adapter.linear(x, w, b, residual=res, act="silu"), want, linear_tol(x, w, b, res, want, dt), (kind, m, k, n))
    wide = torch.randn(m, k + 3, device="cuda", generator=g).to(dt)[:, 1:k + 1]
    want = oa.linear(wide, w)
    close(adapter.linear(wide, w), want, linear_tol(wide, w, None, None, want, dt), "apart")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("t, e, k, d, n", [(4448, 12, 1, 328, 2406), (2273, 3, 3, 136, 2273), (2311, 12, 2, 72, 1436), (1228, 12, 1, 72, 1977),
                                           (501, 12, 1, 176, 1159), (900, 70, 2, 1032, 990), (89, 8, 3, 400, 2002), (3342, 7, 3, 176, 1519), (376, 11, 1, 216, 1462)])
def test_expert_linear_every_tile(kind, t, e, k, d, n):
    g, dt = gen(t + e + d), TYPES[kind]
    r = choose(g, t, e, k, 0.1)
    x, w, b = randn(g, t, d, dtype=dt), randn(g, e, n, d, dtype=dt, scale=d ** -0.5), randn(g, e, n, dtype=dt)
    check_expert(x, w, r, b, rows="tokens", out="slots", what=(kind, t, e, k, d, n))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows, out", [("tokens", "slots"), ("sorted", "sorted")])
@pytest.mark.parametrize("t, e, k, d, n", [(1, 3, 1, 520, 9), (7, 13, 1, 2432, 40), (9, 70, 2, 1032, 17), (40, 8, 4, 1023, 33), (33, 2, 1, 512, 130), (90, 130, 3, 515, 8),
                                           (100, 8, 2, 1032, 70), (60, 4, 1, 2051, 24)])
def test_expert_linear_few_rows(kind, rows, out, t, e, k, d, n):
    g, dt = gen(t + e + d), TYPES[kind]
    for lost in (0.0, 0.4, 1.0):
        r = choose(g, t, e, k, lost)
        x = randn(g, t if rows == "tokens" else t * k, d, dtype=dt)
        w, b = randn(g, e, n, d, dtype=dt, scale=d ** -0.5), randn(g, e, n)
        check_expert(x, w, r, b, act="hsigmoid" if lost else "gelu", rows=rows, out=out, what=(kind, t, e, k, d, n, lost))
    lies = adapter.Routing(r.weights, r.experts, torch.randint(-5, t * k + 5, (t * k,), generator=g, device="cuda", dtype=torch.int32),
                           torch.randint(-9, 2 * t * k + 9, (e + 1,), generator=g, device="cuda", dtype=torch.int32))
    adapter.expert_linear(x, w, lies, b, rows=rows, out=out)
    torch.cuda.synchronize()


@pytest.mark.gpu
@pytest.mark.parametrize("e", [62, 63, 64, 65, 127, 128, 200])
@pytest.mark.parametrize("t, k", [(2, 1), (90, 7), (1500, 3)])
def test_expert_linear_many_experts(e, t, k):
    g = gen(t + e)
    r = choose(g, t, e, k, 0.2)
    x, w, b = randn(g, t, 64, dtype=torch.bfloat16), randn(g, e, 40, 64, dtype=torch.bfloat16, scale=0.125), randn(g, e, 40)
    check_expert(x, w, r, b, act="silu", rows="tokens", out="slots", what=(e, t, k))


@pytest.mark.gpu
def test_expert_linear_nothing():
    r = choose(gen(1), 0, 4, 2)
    assert adapter.expert_linear(torch.zeros(0, 8, device="cuda"), torch.zeros(4, 6, 8, device="cuda"), r, out="slots").shape == (0, 2, 6)


# ---- together ----------------------------------------------------------------------------------------------------------

def block64(a, x):
    """The block by its definition, the types' roundings between the operators in place."""
    def rnd(v, dt):
        return v.to(dt).double()
    h = rnd(oa.norm(x.double(), a.norm, a.pre_weight, a.pre_bias), a.dtype)
    if isinstance(a, adapter.ResidualAdapter):
        y = rnd(oa.linear(rnd(oa.linear(h, a.w1, a.b1, name=a.act), a.dtype), a.w2, a.b2), a.dtype)
    else:
        wt, ex, _, _ = oa.route(oa.linear(h, a.router), a.k, a.score, a.balance, a.groups, a.top_groups)
        ex = ex.to(x.device)
        up = rnd(oa.expert_linear(h, a.w1, ex, a.b1, name=a.act), a.dtype)
        y = oa.weighted(rnd(oa.expert_linear(up, a.w2, ex, a.b2, tokens=False, slots=True), a.dtype), wt.to(x.device).float())
    out = x.double() + a.scale * a.gate.double() * oa.norm(y, a.norm, a.post_weight, a.post_bias)
    return out, oa.norm(out, "l2")


def filled(a, seed):
    g = torch.Generator().manual_seed(seed)
    for name, p in a.named_parameters():
        if name in ("gate", "b1", "b2", "pre_bias", "post_bias"):
            p.copy_(torch.randn(p.shape, generator=g) * 0.5)
        elif name in ("pre_weight", "post_weight"):
            p.copy_(1 + 0.2 * torch.randn(p.shape, generator=g))
    return a.cuda()


def cosines(a, b):
    return torch.nn.functional.cosine_similarity(a.double(), b.double(), dim=-1)


@pytest.mark.gpu
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("n", [1, 3, 70])
@pytest.mark.parametrize("make", [lambda norm: adapter.ResidualAdapter(512, 1024, norm=norm, dtype=torch.float32),
                                  lambda norm: adapter.ExpertAdapter(512, 256, experts=6, k=2, norm=norm, scale=0.5, dtype=torch.float32),
                                  lambda norm: adapter.ExpertAdapter(512, 256, experts=8, k=3, norm=norm, score="sigmoid", groups=4, top_groups=2, dtype=torch.float32)])
def test_blocks(make, norm, n):
    """Whole blocks in f32.  Four roundings of f32 a way and sums of at most 1024 products: 1024 U of rows of size 1 at each of
    three stages, amplified by norms of order 1 (their weights are below 2): 1e-3 is ten times that."""
    torch.manual_seed(5)
    a = filled(make(norm), 7)
    x = randn(gen(n), n, 512)
    want, unit = block64(a, x)
    assert float((a(x).double() - want).abs().max()) < 1e-3
    assert float((a.rows(x).double() - unit).abs().max()) < 2.0 ** -8
    a.gate.zero_()
    assert torch.equal(a(x), x)


@pytest.mark.gpu
def test_block_in_bf16_stays_near():
    """bf16 products: every stage rounds to 2^-8 relative, four stages; cosine loss is half the square of that."""
    torch.manual_seed(6)
    a = filled(adapter.ResidualAdapter(512, 2048), 8)
    x = randn(gen(2), 200, 512)
    want, _ = block64(a, x)
    assert float(cosines(a(x), want).min()) > 1 - 0.5 * (8 * 2.0 ** -8) ** 2


@pytest.mark.gpu
def test_adapter_on_the_framework_s_paths(tmp_path):
    """embed_images and build_from_images with an adapter; a search over the gallery that was built finds every face."""
    import numpy as np
    from face_recognition_amd import gallery, inference, search
    torch.manual_seed(0)
    model = fr.get_network("mobilenetv3_small").cuda().eval()
    a = filled(adapter.ExpertAdapter(512, 256, experts=4, k=2), 9)
    faces = list(np.random.default_rng(3).integers(0, 256, size=(12, 112, 112, 3), dtype=np.uint8))
    plain = inference.embed_images(model, "cuda", faces, batch_size=5)
    got = inference.embed_images(model, "cuda", faces, batch_size=5, adapter=a)
    assert torch.equal(got, torch.cat([a(plain[i:i + 5]) for i in range(0, 12, 5)]))
    built = gallery.build_from_images(model, "cuda", [str(i) for i in range(12)], faces, str(tmp_path / "g"), batch_size=5, adapter=a)
    rows = built.load_rows("cuda")
    assert torch.equal(rows, torch.cat([a.rows(plain[i:i + 5]) for i in range(0, 12, 5)]))
    _, idx = built.matcher("cuda", k=1).search(a.rows(plain))
    # two faces whose rows agree to the last bit of bf16 are both right answers
    assert all(torch.equal(rows[int(i)], rows[j]) or int(i) == j for j, i in enumerate(idx[:, 0].cpu()))


@pytest.mark.gpu
def test_streams_and_graphs():
    """Blocks on two streams at once; two captured graphs replayed in turn with eager work between, every replay checked."""
    torch.manual_seed(1)
    a = filled(adapter.ExpertAdapter(512, 512, experts=8, k=2), 4)
    xs = [randn(gen(40 + i), n, 512) for i, n in enumerate((300, 300, 7, 64))]
    want = [a(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = {}
    for turn in range(3):
        for i, x in enumerate(xs):
            with torch.cuda.stream(streams[i % 2]):
                got[turn, i] = a(x)
    torch.cuda.synchronize()
    for (turn, i), y in got.items():
        assert torch.equal(y, want[i]), (turn, i)
    graphs = []
    for x in xs[1:3]:
        inp = x.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = a.rows(inp)
        graphs.append((g, inp, out))
    for turn in range(4):
        for j, (g, inp, out) in enumerate(graphs):
            new = randn(gen(100 * turn + j), *inp.shape)
            eager = a.rows(new)
            inp.copy_(new)
            g.replay()
            a(xs[0])
            torch.cuda.synchronize()
            assert torch.equal(out, eager), (turn, j)


@pytest.mark.gpu
def test_usual_calls_take_the_short_way_and_answer_the_same(monkeypatch):
    g = gen(77)
    x, w, b, e = randn(g, 9, 64, dtype=torch.bfloat16), randn(g, 40, 64, dtype=torch.bfloat16), randn(g, 40), randn(g, 5, 40, 64, dtype=torch.bfloat16)
    res, slope, logits, lb = randn(g, 9, 40), randn(g, 40), randn(g, 9, 5), randn(g, 5, scale=0.1)
    gates, sw, y3 = [None, randn(g, 64), randn(g, 9, 1), randn(g, 9, 64)], randn(g, 9, 3), randn(g, 9, 3, 64)
    nw, nb = randn(g, 64), randn(g, 64)
    r = adapter.route(logits, 2)
    calls = [lambda: adapter.linear(x, w), lambda: adapter.linear(x.view(3, 3, 64), w, b, act="prelu", slope=slope, residual=res.view(3, 3, 40), out_dtype=torch.float16),
             lambda: adapter.linear(x, w, w.new_zeros(40), act="gelu", residual=res.half()), lambda: adapter.linear(x[0], w, residual=res[0]),
             lambda: adapter.linear(randn(gen(5), 130, 2048), randn(gen(6), 70, 2048)),
             lambda: adapter.route(logits, 3, score="sigmoid", bias=lb, groups=5, top_groups=4, renormalise=False, scale=2), lambda: adapter.route(logits.half(), 1),
             lambda: adapter.route(logits[:0], 2), lambda: adapter.route(randn(gen(8), 700, 40), 4),
             lambda: adapter.expert_linear(x, e, r, act="silu"), lambda: adapter.expert_linear(x, e, r, randn(gen(3), 5, 40), out="slots", out_dtype=torch.float32),
             lambda: adapter.expert_linear(torch.cat([x, x]), e, r, act="prelu", slope=randn(gen(4), 5, 40), rows="sorted")]
    for gate in gates:
        calls += [lambda gate=gate: adapter.block_norm(x, x.float(), norm="layer", weight=nw, bias=nb, gate=gate, gate_act="tanh", scale=0.5),
                  lambda gate=gate: adapter.block_norm(y3, slot_weights=sw, norm="rms", gate=gate, next_norm="layer", next_weight=nw, next_dtype=torch.bfloat16, eps=0)]
    calls += [lambda: adapter.block_norm(x, norm="none", next_norm="l2", out_dtype=torch.float32), lambda: adapter.block_norm(x[0], norm="l2")]
    flat = lambda v: tuple(v) if isinstance(v, tuple) else (v,)
    taken = []

    class Counted:
        def __getattr__(self, name):
            def call(*args):
                v = getattr(real, name)(*args)
                taken.append(v is not None)
                return v
            return call

    class Never:
        def __getattr__(self, name):
            return lambda *args: None

    real = _lib.calls()
    monkeypatch.setattr(_lib, "calls", lambda: Counted())
    short = [flat(c()) for c in calls]
    assert all(taken) and len(taken) == len(calls)
    monkeypatch.setattr(_lib, "calls", lambda: Never())
    for i, (c, got) in enumerate(zip(calls, short)):
        want = flat(c())
        assert len(want) == len(got)
        for a, z in zip(got, want):
            assert a.dtype == z.dtype and a.shape == z.shape and a.stride() == z.stride() and a.device == z.device and torch.equal(a, z), i
            assert not a.requires_grad
    monkeypatch.setattr(_lib, "calls", lambda: Counted())
    taken.clear()
    wide = randn(g, 9, 128, dtype=torch.bfloat16)
    with torch.no_grad():
        adapter.linear(x.clone().requires_grad_(), w)
    with torch.inference_mode():
        y = adapter.linear(x, w)
        assert y.is_inference() and torch.equal(y, short[0][0])
    assert taken == [True, True]
    taken.clear()
    adapter.linear(wide[:, :64], w)
    adapter.linear(x[:0], w)
    adapter.block_norm(x.t().contiguous().t())
    adapter.route(logits.t().contiguous().t(), 2)
    adapter.route(logits, 2, scale=torch.tensor(1.0).numpy()[()].astype("float64"))
    adapter.expert_linear(wide[:, :64], e, r)
    wrong = (lambda: adapter.linear(x, w.float()), lambda: adapter.linear(x, w[:, :63]), lambda: adapter.linear(x, w, b[:39]), lambda: adapter.linear(x, w, act="tanh"),
                lambda: adapter.linear(x, w, act="prelu"), lambda: adapter.linear(x, w, slope=slope), lambda: adapter.linear(x, w, residual=res[:8]),
                lambda: adapter.linear(x, w.cpu()), lambda: adapter.linear(x.double(), w.double()), lambda: adapter.linear(x, w, out_dtype=torch.int32),
                lambda: adapter.linear(x.clone().requires_grad_(), w), lambda: adapter.block_norm(x, norm="max"), lambda: adapter.block_norm(x, weight=nw[:63]),
                lambda: adapter.block_norm(x, norm="l2", weight=nw), lambda: adapter.block_norm(x, gate=randn(g, 9)), lambda: adapter.block_norm(x, x[:8]),
                lambda: adapter.block_norm(x, slot_weights=sw), lambda: adapter.route(logits, 6), lambda: adapter.route(logits, 2, bias=lb.half()),
                lambda: adapter.route(logits, 2, groups=5, top_groups=6), lambda: adapter.route(logits, 2, score="max"),
                lambda: adapter.expert_linear(x[:8], e, r), lambda: adapter.expert_linear(x, e[:4], r), lambda: adapter.expert_linear(x, e, r, randn(g, 40)),
                lambda: adapter.expert_linear(x, e, r, rows="all"))
    for bad in wrong:
        with pytest.raises(RuntimeError, match="fr_hip::"):
            bad()
    assert len(taken) == 6 + len(wrong) and not any(taken)


@pytest.mark.gpu
def test_dispatched_ops_answer_as_the_functions_do():
    """torch.ops.fr_hip goes through the dispatcher, the functions of adapter straight to the implementation."""
    g = gen(50)
    x, w, b = randn(g, 20, 64), randn(g, 48, 64), randn(g, 48)
    o = torch.ops.fr_hip
    assert torch.equal(o.linear(x, w, b, None, None, "gelu", torch.bfloat16), adapter.linear(x, w, b, act="gelu", out_dtype=torch.bfloat16))
    out, nxt = o.block_norm(x, None, None, "rms", None, None, 1e-6, None, "none", 1.0, "l2", None, None, 1e-6, None, torch.bfloat16)
    want = adapter.block_norm(x, next_norm="l2", next_dtype=torch.bfloat16)
    assert torch.equal(out, want[0]) and torch.equal(nxt, want[1])
    out, nxt = o.block_norm(x, None, None, "rms", None, None, 1e-6, None, "none", 1.0, "none", None, None, 1e-6, None, None)
    assert torch.equal(out, adapter.block_norm(x)) and nxt.numel() == 0
    got = o.route(x, 3, "softmax", None, 4, 2, True, 1.0)
    r = adapter.route(x, 3, groups=4, top_groups=2)
    assert all(torch.equal(a, c) for a, c in zip(got, r))
    we = randn(g, 64, 16, 64)
    assert torch.equal(o.expert_linear(x, we, r.order, r.offsets, 3, None, "none", None, "tokens", "slots", None),
                       adapter.expert_linear(x, we, r, out="slots"))


@pytest.mark.gpu
def test_gradients_are_refused_on_the_gpu():
    x = torch.zeros(2, 8, device="cuda", requires_grad=True)
    w = torch.zeros(4, 8, device="cuda")
    with pytest.raises(RuntimeError, match="inference only"):
        adapter.linear(x, w)
    with pytest.raises(RuntimeError, match="inference only"):
        adapter.block_norm(x)
    with torch.no_grad():
        assert adapter.linear(x, w).shape == (2, 4)
