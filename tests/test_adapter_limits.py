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
