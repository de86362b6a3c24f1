"""The front ends of ``pccs_accel.kernels`` that have no autograd node around them, against the nodes: bit for bit."""
import pytest
import torch

import routing_reference as R
from pccs_accel import kernels as K
from pccs_accel.layers import modality_linear
from pccs_accel.routing import combine, dispatch, route_topk, sort_pairs

pytestmark = pytest.mark.gpu


def _normal(g, dev, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype).to(dev)


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
@pytest.mark.parametrize("normalize", [True, False])
def test_router(gpu_device, dtype, normalize):
    g = torch.Generator().manual_seed(1)
    scores, gw = _normal(g, gpu_device, 70, 41, dtype=dtype).requires_grad_(), _normal(g, gpu_device, 70, 6)
    ids, w = route_topk(scores, 6, normalize=normalize)
    ds, = torch.autograd.grad(w, scores, gw)
    ids2, w2, stats = K.route_topk(scores.detach(), 6, normalize=normalize, want_stats=True)
    assert torch.equal(ids, ids2) and torch.equal(w, w2)
    assert torch.equal(ds, K.route_topk_grad(scores.detach(), ids2, w2, stats, gw, normalize=normalize))


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
def test_rows_there_and_back(gpu_device, dtype):
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(-1, 9, (50, 4), generator=g, dtype=torch.int32).to(gpu_device)
    plan = sort_pairs(ids, 9)
    for a, c in zip(plan, K.sort_pairs(ids, 9)):
        assert torch.equal(a, c)
    x, rows, gy = (_normal(g, gpu_device, n, 37, dtype=dtype) for n in (50, 200, 50))
    weights = torch.rand(50, 4, generator=g).to(gpu_device)
    assert torch.equal(dispatch(x, plan), K.dispatch_rows(x, plan.position, plan.offsets))
    assert torch.equal(combine(rows, plan), K.combine_rows(rows, plan.position, plan.offsets))
    leaves = rows.clone().requires_grad_(), weights.clone().requires_grad_()
    y = combine(leaves[0], plan, leaves[1])
    dr, dw = torch.autograd.grad(y, leaves, gy)
    assert torch.equal(y, K.combine_rows(rows, plan.position, plan.offsets, weights))
    for want_r, want_w in ((True, True), (True, False), (False, True)):
        dr2, dw2 = K.combine_rows_grad(rows, gy, plan.position, plan.offsets, weights, want_rows=want_r, want_weights=want_w)
        assert torch.equal(dr, dr2) if want_r else dr2 is None
        assert torch.equal(dw, dw2) if want_w else dw2 is None


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
@pytest.mark.parametrize("act", [None, "relu", "silu"])
def test_layers_of_modalities(gpu_device, dtype, act):
    g = torch.Generator().manual_seed(3)
    offsets = torch.tensor([0, 30, 30, 77, 90], dtype=torch.int32, device=gpu_device)
    x, w, b, r, gy = (_normal(g, gpu_device, *s, dtype=dtype) for s in ((96, 33), (4, 21, 33), (4, 21), (96, 21), (96, 21)))
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    y = modality_linear(leaves[0], offsets, leaves[1], leaves[2], act, leaves[3])
    dx, dw, db, dr = torch.autograd.grad(y, leaves, gy)
    y2, pre = K.linear(x, w, b, act, r, offsets, want_pre=True)
    assert torch.equal(y, y2) and torch.equal(dr, K.linear_mask_rows(gy, offsets))
    for a, c in zip((dx, dw, db), K.linear_backward(gy, pre, act, x, w, offsets)):
        assert torch.equal(a, c)
    want = R.modality_linear(*(t.cpu() for t in (x, offsets, w, b)), act, r.cpu(), gy.cpu())
    dz = K.linear_act_grad(gy, pre, act, offsets) if act else gy  # step by step the tiles may be others
    R.check("dx", K.linear_grad_input(dz, w, offsets), want["dx"])
    for name, v in zip(("dw", "db"), K.linear_grad_weight(dz, x, offsets, want_bias=True)):
        R.check(name, v, want[name])
