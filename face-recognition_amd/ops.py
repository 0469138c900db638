"""PyTorch-ROCm custom ops over the C-ABI of libfr_hip.so.

BASELINE.json's north_star asks for the hot path to be "swapped in through PyTorch-ROCm custom ops
that call HIP kernels over a thin C-ABI layer".  The ops below are registered with ``torch.library``
under the namespace ``fr_hip`` for the CUDA (= ROCm) dispatch key ONLY: calling one with CPU tensors
raises ``NotImplementedError`` from the dispatcher -- there is no CPU fallback.  Each implementation
validates dtype / shape / contiguity, allocates outputs with torch's caching allocator, and makes
exactly one C-ABI call on the current torch stream (include/fr_hip.h names the reference lines each
call replaces).

    torch.ops.fr_hip.embed(x, plan, out_c, out_h, out_w)      model(tensor)        inference.py:121-122
    torch.ops.fr_hip.embed_u8(x, plan, out_c, out_h, out_w)   transform + model    inference.py:98-106,:120-122
    torch.ops.fr_hip.cosine_pairs(a, b, eps, threshold)       similarity formulas  utils/face_utils.py:84-87, evaluate.py:554,:204-206
    torch.ops.fr_hip.l2norm_bf16(x)                           gallery/query rows   (no counterpart)
    torch.ops.fr_hip.topk_search(q, g, k, idx_offset)         1:N search           (no counterpart)
    torch.ops.fr_hip.topk_merge(scores, idx, k)               shard merge          (no counterpart)
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import Dict, Tuple

import torch
from torch.autograd import forward_ad

from . import _lib

_NS = "fr_hip"
_defs = torch.library.Library(_NS, "DEF")
_defs.define("embed(Tensor x, int plan, int out_c, int out_h, int out_w) -> Tensor")
_defs.define("embed_u8(Tensor x, int plan, int out_c, int out_h, int out_w) -> Tensor")
_defs.define("cosine_pairs(Tensor a, Tensor b, float eps, float threshold) -> (Tensor, Tensor)")
_defs.define("l2norm_bf16(Tensor x) -> Tensor")
_defs.define("topk_search(Tensor q, Tensor g, int k, int idx_offset) -> (Tensor, Tensor)")
_defs.define("topk_merge(Tensor scores, Tensor idx, int k) -> (Tensor, Tensor)")
_defs.define("linear(Tensor x, Tensor weight, Tensor? bias, Tensor? slope, Tensor? residual, str act, ScalarType? out_dtype) -> Tensor")
_defs.define("block_norm(Tensor x, Tensor? residual, Tensor? slot_weights, str norm, Tensor? weight, Tensor? bias, float eps, "
             "Tensor? gate, str gate_act, float scale, str next_norm, Tensor? next_weight, Tensor? next_bias, float next_eps, "
             "ScalarType? out_dtype, ScalarType? next_dtype) -> (Tensor, Tensor)")
_defs.define("route(Tensor logits, int k, str score, Tensor? bias, int groups, int top_groups, bool renormalise, float scale) "
             "-> (Tensor, Tensor, Tensor, Tensor)")
_defs.define("expert_linear(Tensor x, Tensor weight, Tensor order, Tensor offsets, int k, Tensor? bias, str act, Tensor? slope, "
             "str rows, str out, ScalarType? out_dtype) -> Tensor")
_impl = torch.library.Library(_NS, "IMPL", "CUDA")
_meta = torch.library.Library(_NS, "IMPL", "Meta")
_autograd = torch.library.Library(_NS, "IMPL", "Autograd")

# (plan handle | 0 for search, device index, stream handle) -> scratch.  Keyed by STREAM as well: two calls enqueued
# on different streams can overlap on the GPU, and a workspace shared between them (the same model on two streams,
# two Matchers) would be written by both at once.  Calls on one stream are ordered, so they share.
# Growth is bounded: at most MAX_STREAM_WORKSPACES streams per (plan, device) keep a workspace; a server that makes streams
# per request evicts the least recently used one (its memory goes back to torch's caching allocator, which hands a block
# only to later allocations of the stream it was allocated on, so kernels still queued on that stream are safe).
# ``drop_stream_workspaces()`` releases them all, or those of one stream.
_workspaces: Dict[Tuple[int, int, int], torch.Tensor] = {}
MAX_STREAM_WORKSPACES = 8


def _stream(dev) -> int:
    return torch.cuda.current_stream(dev).cuda_stream


def _workspace(key: int, dev: torch.device, nbytes: int) -> torch.Tensor:
    k = (key, dev.index, _stream(dev))
    ws = _workspaces.pop(k, None)
    if ws is None or ws.numel() < nbytes:
        ws = None
        peers = [p for p in _workspaces if p[0] == key and p[1] == dev.index]
        for p in peers[:max(0, len(peers) - (MAX_STREAM_WORKSPACES - 1))]:      # dict order = least recently used first
            del _workspaces[p]
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    _workspaces[k] = ws                                                           # (re-)inserted last = most recently used
    return ws


def drop_stream_workspaces(stream: int = -1) -> int:
    """Release the cached workspaces of one stream handle (``torch.cuda.Stream.cuda_stream``), or of every stream
    (-1).  For servers that retire streams; returns the number released."""
    ks = [k for k in _workspaces if stream == -1 or k[2] == stream]
    for k in ks:
        del _workspaces[k]
    return len(ks)


def drop_workspace(plan: int) -> None:
    """Called when a plan is destroyed."""
    for k in [k for k in _workspaces if k[0] == plan]:
        del _workspaces[k]


def _out_shape(n, c, h, w):
    return (n, c) if (h, w) == (1, 1) else (n, c, h, w)


def _embed_any(x, plan, out_c, out_h, out_w, u8):
    x = x.contiguous()
    n = x.shape[0]
    out = torch.empty(_out_shape(n, out_c, out_h, out_w), dtype=torch.float32, device=x.device)
    if n == 0:
        return out
    lib = _lib.lib()
    need = C.c_size_t()
    _lib.check(lib.fr_plan_workspace_bytes(C.c_void_p(plan), n, C.byref(need)), "fr_plan_workspace_bytes")
    ws = _workspace(plan, x.device, need.value)
    fn, name = (lib.fr_embed_u8, "fr_embed_u8") if u8 else (lib.fr_embed, "fr_embed")
    with torch.cuda.device(x.device):
        _lib.check(fn(C.c_void_p(plan), x.data_ptr(), n, out.data_ptr(), ws.data_ptr(), ws.numel(), _stream(x.device)), name)
    return out


def _embed(x, plan, out_c, out_h, out_w):
    if x.dtype != torch.float32 or x.dim() != 4:
        raise RuntimeError("fr_hip::embed: expected a float32 [N,C,H,W] tensor")
    return _embed_any(x, plan, out_c, out_h, out_w, False)


def _embed_u8(x, plan, out_c, out_h, out_w):
    if x.dtype != torch.uint8 or x.dim() != 4 or x.shape[3] != 3:
        raise RuntimeError("fr_hip::embed_u8: expected a uint8 [N,H,W,3] tensor")
    return _embed_any(x, plan, out_c, out_h, out_w, True)


def _cosine_pairs(a, b, eps, threshold):
    if a.dtype != torch.float32 or b.dtype != torch.float32 or a.dim() != 2 or a.shape != b.shape:
        raise RuntimeError("fr_hip::cosine_pairs: expected two float32 [P,d] tensors of equal shape")
    a, b = a.contiguous(), b.contiguous()
    P, d = a.shape
    sim = torch.empty(P, dtype=torch.float32, device=a.device)
    dec = torch.empty(P, dtype=torch.uint8, device=a.device)
    if P:
        with torch.cuda.device(a.device):
            _lib.check(_lib.lib().fr_cosine_pairs(a.data_ptr(), b.data_ptr(), P, d, C.c_float(eps), C.c_double(threshold),
                                                  sim.data_ptr(), dec.data_ptr(), _stream(a.device)), "fr_cosine_pairs")
    return sim, dec.bool()


def _l2norm_bf16(x):
    if x.dtype != torch.float32 or x.dim() != 2:
        raise RuntimeError("fr_hip::l2norm_bf16: expected a float32 [n,d] tensor")
    x = x.contiguous()
    out = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    if x.shape[0]:
        with torch.cuda.device(x.device):
            _lib.check(_lib.lib().fr_l2norm_bf16(x.data_ptr(), out.data_ptr(), x.shape[0], x.shape[1],
                                                 _stream(x.device)), "fr_l2norm_bf16")
    return out


def _topk_search(q, g, k, idx_offset):
    if q.dtype != torch.bfloat16 or g.dtype != torch.bfloat16 or q.dim() != 2 or g.dim() != 2 or q.shape[1] != g.shape[1]:
        raise RuntimeError("fr_hip::topk_search: expected bf16 [Q,d] queries and bf16 [G,d] gallery rows")
    if q.device != g.device:
        raise RuntimeError("fr_hip::topk_search: queries and gallery must be on the same device")
    q, g = q.contiguous(), g.contiguous()
    Q, G, d = q.shape[0], g.shape[0], q.shape[1]
    scores = torch.empty((Q, k), dtype=torch.float32, device=q.device)
    idx = torch.empty((Q, k), dtype=torch.int64, device=q.device)
    if Q == 0:
        return scores, idx
    if G == 0:
        return scores.fill_(float("-inf")), idx.fill_(-1)
    lib = _lib.lib()
    need = C.c_size_t()
    _lib.check(lib.fr_topk_workspace_bytes(Q, G, k, C.byref(need)), "fr_topk_workspace_bytes")
    ws = _workspace(0, q.device, need.value)
    with torch.cuda.device(q.device):
        _lib.check(lib.fr_topk_search(q.data_ptr(), g.data_ptr(), Q, G, d, k, idx_offset, scores.data_ptr(), idx.data_ptr(),
                                      ws.data_ptr(), ws.numel(), _stream(q.device)), "fr_topk_search")
    return scores, idx


def _topk_merge(scores, idx, k):
    if scores.dtype != torch.float32 or idx.dtype != torch.int64 or scores.dim() != 3 or scores.shape != idx.shape \
            or scores.shape[2] != k:
        raise RuntimeError("fr_hip::topk_merge: expected float32 / int64 [P,Q,k] tensors")
    scores, idx = scores.contiguous(), idx.contiguous()
    P, Q, _ = scores.shape
    out_s = torch.empty((Q, k), dtype=torch.float32, device=scores.device)
    out_i = torch.empty((Q, k), dtype=torch.int64, device=scores.device)
    if Q:
        with torch.cuda.device(scores.device):
            _lib.check(_lib.lib().fr_topk_merge(scores.data_ptr(), idx.data_ptr(), P, Q, k, out_s.data_ptr(),
                                                out_i.data_ptr(), _stream(scores.device)), "fr_topk_merge")
    return out_s, out_i


# ---- adapter blocks (adapter.py) ---------------------------------------------------------------------------------------
# Scratch is allocated per call: a call captured into a graph gets memory of the graph's own pool, so two graphs, or a graph
# and the eager program, never write to the same workspace.
_TYPES = {torch.float32: _lib.FR_TYPE_F32, torch.bfloat16: _lib.FR_TYPE_BF16, torch.float16: _lib.FR_TYPE_F16}
_ACTS = {"none": _lib.FR_ACT_NONE, "prelu": _lib.FR_ACT_PRELU, "hswish": _lib.FR_ACT_HSWISH, "relu": _lib.FR_ACT_RELU,
         "hsigmoid": _lib.FR_ACT_HSIGMOID, "gelu": _lib.FR_ACT_GELU, "silu": _lib.FR_ACT_SILU}
_NORMS = {"none": _lib.FR_NORM_NONE, "rms": _lib.FR_NORM_RMS, "layer": _lib.FR_NORM_LAYER, "l2": _lib.FR_NORM_L2}
_GATE_ACTS = {"none": _lib.FR_GATE_NONE, "sigmoid": _lib.FR_GATE_SIGMOID, "tanh": _lib.FR_GATE_TANH}
_SCORES = {"softmax": _lib.FR_SCORE_SOFTMAX, "sigmoid": _lib.FR_SCORE_SIGMOID}
_ROWS = {"tokens": 0, "sorted": 1}
_OUTS = {"sorted": 0, "slots": 1}


def _fail(op, what):
    raise RuntimeError(f"fr_hip::{op}: {what}")


def _name(op, table, key, what):
    code = table.get(key)
    if code is None:
        _fail(op, f"{what} is one of {', '.join(table)}: got {key!r}")
    return code


def _type(op, what, dtype):
    code = _TYPES.get(dtype)
    if code is None:
        _fail(op, f"{what} is float32, bfloat16 or float16: got {dtype}")
    return code


def _no_gradient(op, *tensors):
    """The kernels have no backward pass and carry no tangents, and a result that silently cuts the graph would be a wrong one."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                _fail(op, "inference only: call it under torch.no_grad() or on detached tensors")
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                _fail(op, "inference only: a tensor has a forward-mode tangent")


def _check_tensors(op, first, *others):
    """One device, and no gradient asked for."""
    dev, index = first.device, first.get_device()
    for t in others:
        if t is not None and (t.get_device() != index or (index < 0 and t.device != dev)):
            _fail(op, f"all tensors on {dev}: got one on {t.device}")
    _no_gradient(op, first, *others)
    return dev


def _ptr(t):
    return None if t is None else t.data_ptr()


def _current_device():
    return torch._C._cuda_getDevice()


def _current_stream(index):
    return torch._C._cuda_getCurrentRawStream(index)


def _call(name, dev, *args):
    """One C-ABI call on the device's current stream.  A call on one row takes a few microseconds on the GPU, so the host's
    share counts: no Stream object, no device switch where none is needed."""
    index = dev.index
    fn = _entry(name)
    if _current_device() == index:
        rc = fn(*args, _current_stream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _current_stream(index))
    if rc:
        _lib.check(rc, name)


@functools.lru_cache(maxsize=None)
def _entry(name):
    return getattr(_lib.lib(), name)


@functools.lru_cache(maxsize=1024)
def _scratch_bytes(name, *shape):
    """Workspace of a shape, by shape alone (the rules behind it are the library's, fixed for the process)."""
    need = C.c_size_t()
    _lib.check(getattr(_lib.lib(), name)(*shape, C.byref(need)), name)
    return need.value


def _rows(t, width):
    """``t`` [..., width] as rows: (tensor, row stride).  A matrix whose rows are whole but apart is taken as it lies."""
    if t.is_contiguous():
        return t, width
    if t.dim() == 2 and (t.stride(1) == 1 or width == 1) and t.stride(0) >= 0:
        return t, t.stride(0)
    return t.contiguous(), width


def _check_of(op, what, t, shape, *dtypes):
    if t.shape != shape or t.dtype not in dtypes:
        _fail(op, f"{what} is {list(shape)} of {' or '.join(str(d)[6:] for d in dtypes)}: got {t.dtype} {tuple(t.shape)}")


def _whole(t):
    return None if t is None else t.contiguous()


# The checks of an operator's arguments, of tensors with and without data alike.
def _check_linear(x, weight, bias, slope, residual, act, out_dtype):
    """(device, shape of the result, codes of x's type, of out_dtype and of act)."""
    op = "linear"
    dev = _check_tensors(op, x, weight, bias, slope, residual)
    xs, ws = x.shape, weight.shape
    if len(xs) < 1 or len(ws) != 2 or xs[-1] != ws[1] or ws[1] < 1 or ws[0] < 1:
        _fail(op, f"expected x [..., K] and weight [N, K]: got {tuple(xs)} and {tuple(ws)}")
    if max(ws) >= 1 << 31:
        _fail(op, f"N and K have to fit 31 bits: got {tuple(ws)}")
    shape = xs[:-1] + ws[:1]
    if residual is not None and residual.shape != shape:
        _fail(op, f"residual is {tuple(shape)}: got {tuple(residual.shape)}")
    kind, code = _check_product(op, x, weight, bias, slope, ws[:1], act)
    if residual is not None:
        _type(op, "residual", residual.dtype)
    return dev, shape, kind, kind if out_dtype is None else _type(op, "out_dtype", out_dtype), code


def _check_product(op, x, weight, bias, slope, shape, act):
    """What the two products have in common: (code of x's type, of act)."""
    kind = _type(op, "x", x.dtype)
    if weight.dtype != x.dtype:
        _fail(op, f"x and weight have one type: got {x.dtype} and {weight.dtype}")
    code = _name(op, _ACTS, act, "act")
    if (slope is not None) != (code == _lib.FR_ACT_PRELU):
        _fail(op, "slope belongs to act='prelu', and only to it")
    if bias is not None:
        _check_of(op, "bias", bias, shape, x.dtype, torch.float32)
    if slope is not None:
        _check_of(op, "slope", slope, shape, torch.float32)
    return kind, code


# Each of the four first offers its call to csrc/calls.cpp, which takes the usual ones (plain contiguous tensors on the current
# device) with a third of the host's time; the rest, and every wrong one, is dealt with here.  ``way`` says where the call comes from.
# _DIRECT: not through the dispatcher; where that has something to do (csrc/calls.cpp says NotImplemented) it goes there.
# _ABOVE: the dispatcher, before autograd; no answer (None) unless the short way has one.  _BELOW: the dispatcher, as the kernel.
_DIRECT, _ABOVE, _BELOW = 0, 1, 2


def _linear(x, weight, bias, slope, residual, act, out_dtype, way=_DIRECT):
    if x.is_cuda:
        index = _current_device()
        y = _lib.calls().linear(x, weight, bias, slope, residual, _ACTS.get(act, -1), out_dtype, index, _current_stream(index))
        if y is not None and y is not NotImplemented:
            return y
        if y is NotImplemented and way == _DIRECT:
            return torch.ops.fr_hip.linear(x, weight, bias, slope, residual, act, out_dtype)
    if way == _ABOVE:
        return None
    dev, shape, kind, out_type, code = _check_linear(x, weight, bias, slope, residual, act, out_dtype)
    N, K = weight.shape
    out = x.new_empty(shape) if out_dtype is None else x.new_empty(shape, dtype=out_dtype)
    M = out.numel() // N
    if M == 0:
        return out
    x, ldx = _rows(x, K)
    weight, bias, slope = weight.contiguous(), _whole(bias), _whole(slope)
    res_type, ldr = kind, 0
    if residual is not None:
        res_type = _TYPES[residual.dtype]
        residual, ldr = _rows(residual, N)
    need = _scratch_bytes("fr_linear_workspace_bytes", M, N, K, kind)
    ws = x.new_empty(need, dtype=torch.uint8) if need else None
    _call("fr_linear", dev, x.data_ptr(), ldx, weight.data_ptr(), _ptr(bias), _ptr(slope), _ptr(residual), ldr, out.data_ptr(),
          M, N, K, kind, kind if bias is None else _TYPES[bias.dtype], res_type, out_type, code, _ptr(ws), need)
    return out


def _check_block_norm(x, residual, slot_weights, norm, weight, bias, gate, gate_act, next_norm, next_weight, next_bias, out_dtype, next_dtype):
    """(device, shape of the results, their dtypes, the gate's strides along rows and columns, codes of norm, next_norm and gate_act)."""
    op = "block_norm"
    dev = _check_tensors(op, x, residual, slot_weights, weight, bias, gate, next_weight, next_bias)
    if x.dim() < (1 if slot_weights is None else 2) or x.shape[-1] < 1:
        _fail(op, f"expected x [..., d], or [..., slots, d] with slot_weights: got {tuple(x.shape)}")
    d, shape = x.shape[-1], x.shape
    if d > 16384:
        _fail(op, f"d is at most 16384: got {d}")
    if slot_weights is not None:
        if x.shape[-2] >= 1 << 31:
            _fail(op, "slots have to fit 31 bits")
        if slot_weights.shape != x.shape[:-1] or slot_weights.dtype != torch.float32 or x.shape[-2] < 1:
            _fail(op, f"slot_weights is float32 {tuple(x.shape[:-1])}: got {slot_weights.dtype} {tuple(slot_weights.shape)}")
        shape = x.shape[:-2] + x.shape[-1:]
    norm, next_norm = _name(op, _NORMS, norm, "norm"), _name(op, _NORMS, next_norm, "next_norm")
    for what, code, w, b in (("", norm, weight, bias), ("next_", next_norm, next_weight, next_bias)):
        if (w is not None or b is not None) and code not in (_lib.FR_NORM_RMS, _lib.FR_NORM_LAYER):
            _fail(op, f"{what}weight and {what}bias belong to the rms and layer norms")
        if w is not None:
            _check_of(op, what + "weight", w, (d,), torch.float32)
        if b is not None:
            _check_of(op, what + "bias", b, (d,), torch.float32)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    next_dtype = out_dtype if next_dtype is None else next_dtype
    for what, dtype in (("out_dtype", out_dtype), ("next_dtype", next_dtype), ("x", x.dtype)):
        _type(op, what, dtype)
    if residual is not None:
        if residual.shape != shape:
            _fail(op, f"residual is {tuple(shape)}: got {tuple(residual.shape)}")
        _type(op, "residual", residual.dtype)
    strides = 0, 0
    if gate is not None:
        _type(op, "gate", gate.dtype)
        if gate.shape == (d,):
            strides = 0, 1
        elif gate.shape == shape:
            strides = d, 1
        elif gate.shape == shape[:-1] + (1,):
            strides = 1, 0
        else:
            _fail(op, f"gate is [{d}], {tuple(shape[:-1]) + (1,)} or {tuple(shape)}: got {tuple(gate.shape)}")
    return dev, shape, out_dtype, next_dtype, strides, norm, next_norm, _name(op, _GATE_ACTS, gate_act, "gate_act")


def _block_norm_eager(x, residual, slot_weights, norm, weight, bias, eps, gate, gate_act, scale, next_norm, next_weight, next_bias,
                      next_eps, out_dtype, next_dtype, way=_DIRECT):
    """(out, next), None (through the dispatcher: a tensor without elements) for a next that is not asked for."""
    if x.is_cuda:
        index = _current_device()
        both = _lib.calls().block_norm(x, residual, slot_weights, _NORMS.get(norm, -1), weight, bias, eps, gate, _GATE_ACTS.get(gate_act, -1),
                                       scale, _NORMS.get(next_norm, -1), next_weight, next_bias, next_eps, out_dtype, next_dtype,
                                       index, _current_stream(index))
        if both is not None and both is not NotImplemented:
            return both
        if both is NotImplemented and way == _DIRECT:
            return torch.ops.fr_hip.block_norm(x, residual, slot_weights, norm, weight, bias, eps, gate, gate_act, scale, next_norm,
                                               next_weight, next_bias, next_eps, out_dtype, next_dtype)
    if way == _ABOVE:
        return None
    dev, shape, out_dtype, next_dtype, (gate_ldt, gate_ldc), norm, next_norm, gate_act = _check_block_norm(
        x, residual, slot_weights, norm, weight, bias, gate, gate_act, next_norm, next_weight, next_bias, out_dtype, next_dtype)
    d = x.shape[-1]
    out = x.new_empty(shape, dtype=out_dtype)
    nxt = x.new_empty(shape, dtype=next_dtype) if next_norm else None
    T = out.numel() // d
    if T == 0:
        return out, nxt
    slots = 0 if slot_weights is None else x.shape[-2]
    x, residual, slot_weights, weight, bias, gate, next_weight, next_bias = map(_whole, (x, residual, slot_weights, weight, bias, gate, next_weight, next_bias))
    _call("fr_block_norm", dev, x.data_ptr(), _TYPES[x.dtype], slots, _ptr(slot_weights), T, d, norm, _ptr(weight), _ptr(bias), eps,
          _ptr(gate), 0 if gate is None else _TYPES[gate.dtype], gate_ldt, gate_ldc, gate_act, scale,
          _ptr(residual), 0 if residual is None else _TYPES[residual.dtype], out.data_ptr(), _TYPES[out_dtype],
          next_norm, _ptr(next_weight), _ptr(next_bias), next_eps, _ptr(nxt), _TYPES[next_dtype])
    return out, nxt


def _block_norm(x, residual, slot_weights, norm, weight, bias, eps, gate, gate_act, scale, next_norm, next_weight, next_bias,
                next_eps, out_dtype, next_dtype, way=_DIRECT):
    both = _block_norm_eager(x, residual, slot_weights, norm, weight, bias, eps, gate, gate_act, scale, next_norm, next_weight,
                             next_bias, next_eps, out_dtype, next_dtype, way)
    if both is None:
        return None
    out, nxt = both
    return out, x.new_empty(0, dtype=next_dtype or out.dtype) if nxt is None else nxt      # the op's schema has two results


def _check_route(logits, k, score, bias, groups, top_groups):
    """(device, codes of the logits' type and of score)."""
    op = "route"
    dev = _check_tensors(op, logits, bias)
    if logits.dim() != 2 or logits.shape[1] < 1:
        _fail(op, f"expected logits [T, E]: got {tuple(logits.shape)}")
    E = logits.shape[1]
    if E > 512:
        _fail(op, f"at most 512 experts: got {E}")
    if not 1 <= k <= min(E, 16):
        _fail(op, f"1 <= k <= 16 of {E} experts: got {k}")
    if logits.shape[0] >= 1 << 30 or logits.shape[0] * k >= 1 << 31:
        _fail(op, f"T has to fit 30 bits and T * k 31: got {logits.shape[0]} and k = {k}")
    if not 1 <= groups <= 64 or not 1 <= top_groups <= groups or E % groups:
        _fail(op, f"1 <= top_groups <= groups <= 64, groups dividing {E}: got {top_groups} of {groups}")
    if top_groups * (E // groups) < k:
        _fail(op, f"{top_groups} of {groups} groups hold fewer than {k} experts")
    kind = _type(op, "logits", logits.dtype)
    if bias is not None:
        _check_of(op, "bias", bias, (E,), torch.float32)
    return dev, kind, _name(op, _SCORES, score, "score")


def _route_empty(logits, k):
    T, E = logits.shape
    i32 = torch.int32
    return (logits.new_empty((T, k), dtype=torch.float32), logits.new_empty((T, k), dtype=i32), logits.new_empty(T * k, dtype=i32),
            logits.new_empty(E + 1, dtype=i32))


def _route(logits, k, score, bias, groups, top_groups, renormalise, scale, way=_DIRECT):
    if logits.is_cuda:
        index = _current_device()
        out = _lib.calls().route(logits, k, _SCORES.get(score, -1), bias, groups, top_groups, renormalise, scale, index, _current_stream(index))
        if out is not None and out is not NotImplemented:
            return out
        if out is NotImplemented and way == _DIRECT:
            return torch.ops.fr_hip.route(logits, k, score, bias, groups, top_groups, renormalise, scale)
    if way == _ABOVE:
        return None
    dev, kind, score = _check_route(logits, k, score, bias, groups, top_groups)
    T, E = logits.shape
    logits, bias = logits.contiguous(), _whole(bias)
    need = _scratch_bytes("fr_route_workspace_bytes", T, E, k)
    out = _route_empty(logits, k)
    ws = logits.new_empty(need, dtype=torch.uint8) if need else None
    _call("fr_route", dev, logits.data_ptr(), kind, T, E, k, score, _ptr(bias), groups, top_groups, renormalise, scale,
          out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), out[3].data_ptr(), _ptr(ws), need)
    return out


def _check_expert_linear(x, weight, order, offsets, k, bias, act, slope, rows, out, out_dtype):
    """(device, shape of the result, codes of x's type, of out_dtype and of act)."""
    op = "expert_linear"
    dev = _check_tensors(op, x, weight, order, offsets, bias, slope)
    if x.dim() != 2 or weight.dim() != 3 or x.shape[1] != weight.shape[2] or min(weight.shape) < 1:
        _fail(op, f"expected x [rows, K] and weight [E, N, K]: got {tuple(x.shape)} and {tuple(weight.shape)}")
    if rows not in ("tokens", "sorted") or out not in ("sorted", "slots"):
        _fail(op, f"rows is 'tokens' or 'sorted', out 'sorted' or 'slots': got {rows!r}, {out!r}")
    if order.dtype != torch.int32 or offsets.dtype != torch.int32 or order.dim() != 1 or offsets.shape != (weight.shape[0] + 1,):
        _fail(op, f"expected int32 order [T*k] and offsets [{weight.shape[0] + 1}] as route returns them")
    if k < 1 or order.shape[0] % k or order.shape[0] >= 1 << 31:
        _fail(op, f"{order.shape[0]} slots are no multiple of k = {k} below 2^31")
    if max(weight.shape) >= 1 << 31:
        _fail(op, f"E, N and K have to fit 31 bits: got {tuple(weight.shape)}")
    T = order.shape[0] // k
    if x.shape[0] != (T if rows == "tokens" else T * k):
        _fail(op, f"rows={rows!r} takes {T if rows == 'tokens' else T * k} rows of x: got {x.shape[0]}")
    kind, code = _check_product(op, x, weight, bias, slope, weight.shape[:2], act)
    shape = (T * k, weight.shape[1]) if out == "sorted" else (T, k, weight.shape[1])
    return dev, shape, kind, kind if out_dtype is None else _type(op, "out_dtype", out_dtype), code


def _expert_linear(x, weight, order, offsets, k, bias, act, slope, rows, out, out_dtype, way=_DIRECT):
    if x.is_cuda:
        index = _current_device()
        y = _lib.calls().expert_linear(x, weight, order, offsets, k, bias, _ACTS.get(act, -1), slope, _ROWS.get(rows, -1), _OUTS.get(out, -1),
                                       out_dtype, index, _current_stream(index))
        if y is not None and y is not NotImplemented:
            return y
        if y is NotImplemented and way == _DIRECT:
            return torch.ops.fr_hip.expert_linear(x, weight, order, offsets, k, bias, act, slope, rows, out, out_dtype)
    if way == _ABOVE:
        return None
    dev, shape, kind, out_type, code = _check_expert_linear(x, weight, order, offsets, k, bias, act, slope, rows, out, out_dtype)
    E, N, K = weight.shape
    y = x.new_empty(shape) if out_dtype is None else x.new_empty(shape, dtype=out_dtype)
    T = order.shape[0] // k
    if T == 0:
        return y
    x, weight, order, offsets, bias, slope = map(_whole, (x, weight, order, offsets, bias, slope))
    _call("fr_expert_linear", dev, x.data_ptr(), int(rows == "sorted"), weight.data_ptr(), _ptr(bias), _ptr(slope), order.data_ptr(),
          offsets.data_ptr(), y.data_ptr(), int(out == "slots"), T, k, E, N, K, kind, kind if bias is None else _TYPES[bias.dtype],
          out_type, code)
    return y


_impl.impl("embed", _embed)
_impl.impl("embed_u8", _embed_u8)
_impl.impl("cosine_pairs", _cosine_pairs)
_impl.impl("l2norm_bf16", _l2norm_bf16)
_impl.impl("topk_search", _topk_search)
_impl.impl("topk_merge", _topk_merge)


def _register(name, impl):
    """The kernel, and above it, for the calls that the short way does not take, the refusal of gradients: it has to stand where
    the dispatcher still sees them, as below autograd a transform's tensors (torch.func.grad, jvp) have neither gradient nor tangent."""
    op = getattr(torch.ops.fr_hip, name).default

    def above(keys, *args):
        if type(args[0]) is torch.Tensor:                     # nothing that only stands in for one
            out = impl(*args, _ABOVE)
            if out is not None:
                return out
        _no_gradient(name, *(a for a in args if isinstance(a, torch.Tensor)))
        with torch._C._AutoDispatchBelowAutograd():
            return op.redispatch(keys & torch._C._after_autograd_keyset, *args)

    _autograd.impl(name, above, with_keyset=True)
    _impl.impl(name, lambda *args: impl(*args, _BELOW))


for _name_impl in (("linear", _linear), ("block_norm", _block_norm), ("route", _route), ("expert_linear", _expert_linear)):
    _register(*_name_impl)

# shape functions (tracing / torch.export)
_meta.impl("embed", lambda x, plan, c, h, w: x.new_empty(_out_shape(x.shape[0], c, h, w), dtype=torch.float32))
_meta.impl("embed_u8", lambda x, plan, c, h, w: x.new_empty(_out_shape(x.shape[0], c, h, w), dtype=torch.float32))
_meta.impl("cosine_pairs", lambda a, b, eps, thr: (a.new_empty(a.shape[0], dtype=torch.float32),
                                                   a.new_empty(a.shape[0], dtype=torch.bool)))
_meta.impl("l2norm_bf16", lambda x: x.new_empty(x.shape, dtype=torch.bfloat16))
_meta.impl("topk_search", lambda q, g, k, off: (q.new_empty((q.shape[0], k), dtype=torch.float32),
                                                q.new_empty((q.shape[0], k), dtype=torch.int64)))
_meta.impl("topk_merge", lambda s, i, k: (s.new_empty((s.shape[1], k), dtype=torch.float32),
                                          s.new_empty((s.shape[1], k), dtype=torch.int64)))


def _meta_linear(x, weight, bias, slope, residual, act, out_dtype):
    return x.new_empty(_check_linear(x, weight, bias, slope, residual, act, out_dtype)[1], dtype=out_dtype or x.dtype)


def _meta_block_norm(x, residual, slot_weights, norm, weight, bias, eps, gate, gate_act, scale, next_norm, next_weight, next_bias,
                     next_eps, out_dtype, next_dtype):
    _, shape, out_dtype, next_dtype, *_ = _check_block_norm(x, residual, slot_weights, norm, weight, bias, gate, gate_act, next_norm, next_weight,
                                                            next_bias, out_dtype, next_dtype)
    return x.new_empty(shape, dtype=out_dtype), x.new_empty(shape if next_norm != "none" else 0, dtype=next_dtype)


def _meta_route(logits, k, score, bias, groups, top_groups, renormalise, scale):
    _check_route(logits, k, score, bias, groups, top_groups)
    return _route_empty(logits, k)


def _meta_expert_linear(x, weight, order, offsets, k, bias, act, slope, rows, out, out_dtype):
    return x.new_empty(_check_expert_linear(x, weight, order, offsets, k, bias, act, slope, rows, out, out_dtype)[1], dtype=out_dtype or x.dtype)


_meta.impl("linear", _meta_linear)
_meta.impl("block_norm", _meta_block_norm)
_meta.impl("route", _meta_route)
_meta.impl("expert_linear", _meta_expert_linear)
