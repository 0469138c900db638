"""Adapter operators at the limits of what their documentation allows: group sums that cancel, biases without bound, tables
that lie, counts that overflow.  Choices are compared as whole numbers; the tolerances of weights are those of test_adapter."""
import math

import pytest
import torch

from face_recognition_amd import adapter
from oracle import adapter as oa
from test_adapter import check_route, gen, randn


# ---- route -------------------------------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("big", [10.0, 100.0, 1e4])
@pytest.mark.parametrize("e, groups, top, k", [(4, 2, 1, 2), (16, 4, 2, 3), (64, 8, 3, 4), (96, 3, 1, 5)])
def test_route_groups_whose_best_two_cancel(score, big, e, groups, top, k):
    """Biases of both signs: the sum of a group's best two keys is small and its error is that of the keys."""
    g, per = gen(e + int(big)), e // groups
    sign = torch.full((groups, per), -2.0, device="cuda")
    sign[:, 0], sign[:, 1] = 1.0, -1.0                         # the best two of every group: one up, one down by the same
    bias = (sign * big).reshape(-1)
    apart = randn(g, 400, e)
    # groups of the same logits but for a little: sums next to each other
    near = randn(g, 400, 1, per).expand(400, groups, per).reshape(400, e) + randn(g, 400, e, scale=big * 2.0 ** -23)
    for what, logits in (("apart", apart), ("near", near)):
        check_route(logits, k, score=score, bias=bias, groups=groups, top_groups=top, what=(what, score, big, e))
    # the large keys in some groups only: their error is no reason to doubt the others, and is one where they stand at the cut
    mixed = torch.where(torch.arange(e, device="cuda") < e // 2, bias, randn(g, e, scale=0.1))
    check_route(apart, k, score=score, bias=mixed, groups=groups, top_groups=top, what=("mixed", score, big, e))


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("kind", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("e, groups, top, k", [(8, 4, 2, 3), (64, 8, 3, 6), (100, 5, 4, 2)])
def test_route_bias_of_infinity_in_groups(score, kind, e, groups, top, k):
    """+inf puts an expert first; alone in its group it leaves the group without a best two, as any other bias does."""
    g, per = gen(e), e // groups
    logits = randn(g, 70, e, dtype=kind)
    bias = randn(g, e, scale=0.1)
    bias[1], bias[per + 1] = math.inf, math.inf
    logits[::2, 0], logits[::2, 2:per] = -math.inf, -math.inf  # expert 1 is alone in its group
    logits[5, per + 1] = math.nan
    got = adapter.route(logits, k, score=score, bias=bias, groups=groups, top_groups=top)
    for r in range(70):
        chosen = {x // per for x in got.experts[r].tolist() if x >= 0}
        assert len(chosen) <= top
    finite = bias.clone()
    finite[1], finite[per + 1] = 2e6, 1e6                      # the same order: scores are at most 1, the lower of two infinities first
    alone = finite.clone()
    alone[1] = 0.0                                             # the sum of a lone expert is -inf whatever its bias
    for rows, b in ((slice(0, None, 2), alone), (slice(1, None, 2), finite)):
        w, ex, _, _ = oa.route(logits[rows], k, score, b, groups, top)
        assert torch.equal(got.experts[rows].cpu(), ex), rows
        assert float((got.weights[rows].cpu().double() - w).abs().max()) < (128 + e) * 2.0 ** -24


# ---- expert_linear -----------------------------------------------------------------------------------------------------

def expert_entry(x, w, order, offsets, k, rows_sorted, out_slots, out):
    """The C entry, into memory of the caller's."""
    from face_recognition_amd import _lib, ops
    E, N, K = w.shape
    _lib.check(_lib.lib().fr_expert_linear(x.data_ptr(), rows_sorted, w.data_ptr(), None, None, order.data_ptr(), offsets.data_ptr(), out.data_ptr(), out_slots,
                                           order.numel() // k, k, E, N, K, ops._TYPES[x.dtype], ops._TYPES[x.dtype], ops._TYPES[out.dtype], 0,
                                           torch.cuda.current_stream().cuda_stream), "fr_expert_linear")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows_sorted, out_slots", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("t, e, k, d, n", [(5, 8, 2, 512, 40), (9, 70, 2, 515, 17), (300, 3, 2, 65, 70), (300, 3, 2, 128, 70), (1500, 2, 2, 256, 264), (4000, 2, 1, 65, 520)])
def test_expert_linear_order_entries_that_lie_are_skipped(kind, rows_sorted, out_slots, t, e, k, d, n):
    """Few rows, rows of any alignment, small and large tiles: nothing is written for such an entry, and nothing outside the output."""
    g, P, MARK = gen(t + d), t * k, 7.0
    ex = torch.randint(0, e, (t, k), generator=g, device="cuda", dtype=torch.int32)
    ex[torch.rand(t, k, generator=g, device="cuda") < 0.2] = -1
    order, offsets = oa.routing_of(ex, e)
    x, w = randn(g, P if rows_sorted else t, d, dtype=kind), randn(g, e, n, d, dtype=kind)
    room = 4096

    def run(order):
        memory = torch.full((2 * room + P * n,), MARK, dtype=kind, device="cuda")
        out = memory[room:room + P * n]
        expert_entry(x, w, order, offsets, k, rows_sorted, out_slots, out)
        torch.cuda.synchronize()
        assert (memory[:room] == MARK).all() and (memory[-room:] == MARK).all()
        return out.view(P, n)

    want = run(order)
    lies = order.clone()
    at = torch.randperm(P, generator=g, device="cuda")[:max(2, P // 7)]
    lies[at] = torch.tensor([P, -1, 1 << 30, -(1 << 31)], device="cuda", dtype=torch.int32)[torch.arange(at.numel(), device="cuda") % 4]
    if out_slots:
        want[order[at].long()] = MARK
    elif not rows_sorted:
        want[at] = MARK
    assert torch.equal(run(lies), want)


@pytest.mark.gpu
@pytest.mark.parametrize("t, e, k, d, n", [(5, 8, 2, 512, 40), (9, 70, 2, 515, 17), (300, 3, 2, 65, 70), (1500, 2, 2, 256, 264)])
def test_expert_linear_offsets_that_lie_write_nothing_outside(t, e, k, d, n):
    g, P, MARK, room = gen(t + d), t * k, 7.0, 4096
    x, w = randn(g, t, d, dtype=torch.bfloat16), randn(g, e, n, d, dtype=torch.bfloat16)
    order = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    for _ in range(6):
        offsets = torch.randint(-P, 3 * P, (e + 1,), generator=g, device="cuda", dtype=torch.int32)
        memory = torch.full((2 * room + P * n,), MARK, dtype=torch.bfloat16, device="cuda")
        expert_entry(x, w, order, offsets, k, 0, 0, memory[room:room + P * n])
        torch.cuda.synchronize()
        assert (memory[:room] == MARK).all() and (memory[-room:] == MARK).all()


# ---- counts that wrap --------------------------------------------------------------------------------------------------

def test_c_entries_refuse_counts_that_wrap():
    """Row counts whose products leave 64 bits are refused before anything is launched (there is no GPU here)."""
    import ctypes as C
    from face_recognition_amd import _lib
    lib, at, need = _lib.lib(), 4096, C.c_size_t()

    def refused(rc, words):
        assert rc == -2 and words in lib.fr_last_error().decode(), (rc, lib.fr_last_error())

    for T, k in ((1 << 30, 2), ((1 << 33) + 1, (1 << 31) - 1), (1 << 62, 4), ((1 << 62) + 1, 4), ((1 << 63) - 1, 2), ((1 << 61) + 5, 8)):
        refused(lib.fr_expert_linear(at, 0, at, None, None, at, at, at, 0, T, k, 4, 8, 8, 1, 1, 1, 0, None), "31 bits")
    for M in (1 << 40, 1 << 57, (1 << 63) - 1):
        refused(lib.fr_linear(at, 8, at, None, None, None, 0, at, M, 8, 8, 1, 1, 1, 1, 0, None, 0, None), "40 bits")
        refused(lib.fr_linear_workspace_bytes(M, 8, 4096, 1, C.byref(need)), "40 bits")
        refused(lib.fr_block_norm(at, 1, 0, None, M, 8, 1, None, None, 1e-6, None, 1, 0, 1, 0, 1.0, None, 0, at, 1, 0, None, None, 1e-6, None, 1, None), "40 bits")
