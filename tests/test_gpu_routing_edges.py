"""``pccs_accel.routing`` where a call can go wrong: gradients at places without a choice, plans that name rows which are not there."""
import math

import pytest
import torch

import routing_reference as R
from pccs_accel.routing import PairPlan, combine, dispatch, route_topk, sort_pairs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("normalize", [True, False])
def test_gradients_where_there_is_no_choice_may_hold_anything(gpu_device, normalize):
    """The weight at an id of -1 is the constant 0: a NaN or an infinity there (a loss of its logarithm) says nothing."""
    for dtype in R.TYPES:
        for n in (7, 1100):
            g = torch.Generator().manual_seed(n)
            scores = (torch.randn(n, 30, generator=g) * 2).to(dtype)
            scores[0] = -math.inf
            scores[1, 3:] = -math.inf
            scores[4, 1:] = -math.inf
            gw = torch.randn(n, 9, generator=g)
            want = R.route(scores, 9, normalize, gw)
            assert (want["ids"] < 0).sum() == 9 + 6 + 8
            gw = torch.where(want["ids"] < 0, torch.tensor([math.nan, math.inf, -math.inf])[torch.arange(9) % 3].expand(n, 9), gw)
            leaf = scores.to(gpu_device).requires_grad_()
            ids, w = route_topk(leaf, 9, normalize=normalize)
            ds, = torch.autograd.grad(w, leaf, gw.to(gpu_device))
            assert torch.equal(ids.cpu(), want["ids"])
            R.check("ds", ds, want["ds"])
