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


@pytest.mark.parametrize("d", [3, 8, 24, 40, 136, 600])
def test_places_that_are_none_are_left_out(gpu_device, d):
    """Places below 0 and behind the last row: the pair is not copied, not summed, and has no gradient."""
    n, k = 50, 5
    g = torch.Generator().manual_seed(d)
    plan = sort_pairs(torch.randint(0, 7, (n, k), generator=g, dtype=torch.int32).to(gpu_device), 7)
    wrong = torch.rand(n, k, generator=g) < 0.3
    there = (~wrong).double()
    here = plan.position.cpu().long()
    values = torch.tensor([-1, n * k, n * k + 1, -2 ** 31, 2 ** 31 - 1, -n * k], dtype=torch.int32)
    position = torch.where(wrong, values[torch.arange(n * k).view(n, k) % 6], plan.position.cpu())
    bad = PairPlan(plan.offsets, plan.order, position.to(gpu_device))
    for dtype in R.TYPES:
        u = R.half_step(dtype)
        x, rows, gy = (torch.randn(m, d, generator=g).to(dtype) for m in (n, n * k, n))
        w = torch.rand(n, k, generator=g)
        out = dispatch(x.to(gpu_device), bad).cpu()
        assert torch.equal(out[here[~wrong]], x[:, None].expand(n, k, d)[~wrong])
        leaves = rows.to(gpu_device).requires_grad_(), w.to(gpu_device).requires_grad_()
        y = combine(leaves[0], bad, leaves[1])
        terms = rows.double()[here] * (w.double() * there)[:, :, None]
        v, e = terms.sum(1), (k + 2) * R.U32 * terms.abs().sum(1)
        R.check("y", y, (v, e + u * (v.abs() + e) + R.floor_of(dtype)))
        dr, dw = torch.autograd.grad(y, leaves, gy.to(gpu_device))
        back = w.double()[:, :, None] * gy.double()[:, None]
        R.check("drows", dr[here[~wrong].to(gpu_device)], (back[~wrong], (u + 2 * R.U32) * back[~wrong].abs() + R.floor_of(dtype)))
        prod = rows.double()[here] * gy.double()[:, None] * there[:, :, None]
        R.check("dw", dw, (prod.sum(2), (d + 2) * R.U32 * prod.abs().sum(2)))


def test_sort_of_many_pairs_over_many_modalities(gpu_device):
    """Runs longer than usual, so that their counts do not outgrow the pairs."""
    n, k, e = 4_700_000, 2, 4096
    g = torch.Generator(device=gpu_device).manual_seed(1)
    ids = torch.randint(-1, e, (n, k), generator=g, dtype=torch.int32, device=gpu_device)
    plan = sort_pairs(ids, e)
    key = ids.reshape(-1).long()
    key = torch.where(key < 0, e, key)
    order = torch.sort(key, stable=True).indices
    assert torch.equal(plan.order.long(), order)
    assert torch.equal(plan.position.reshape(-1)[order].long(), torch.arange(n * k, device=gpu_device))
    assert torch.equal(plan.offsets.long(), torch.searchsorted(key[order], torch.arange(e + 1, device=gpu_device)))
