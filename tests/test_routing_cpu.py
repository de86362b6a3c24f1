"""CPU-side checks of the routing and layer entry points: bad arguments are refused on the host before any launch, workspaces
are as large as said, and the plain formulas the GPU tests compare with agree with torch's autograd in float64."""
import math

import pytest
import torch

import routing_reference as R
from pccs_accel import _lib
from pccs_accel import kernels as K
from pccs_accel.layers import linear, modality_linear
from pccs_accel.routing import combine, dispatch, route_topk, sort_pairs

ONE = 4096  # any non-null address: none of these calls gets as far as a launch


def _refused(rc, text):
    assert rc == -1 and text in _lib.lib().mtp_last_error(), (rc, _lib.lib().mtp_last_error())


def test_entry_points_refuse_bad_shapes():
    L = _lib.lib()
    for dtype, n, e, ld, k in ((0, -1, 8, 8, 2), (0, 4, 0, 8, 1), (0, 4, 4097, 4097, 2), (0, 4, 8, 8, 9), (0, 4, 8, 7, 2), (0, 4, 200, 200, 129)):
        _refused(L.mtp_route_topk(dtype, ONE, n, e, ld, k, 0, ONE, ONE, None, None), b"bad shape")
        _refused(L.mtp_route_topk_grad(dtype, ONE, n, e, ld, k, 0, ONE, ONE, ONE, ONE, ONE, None), b"bad shape")
    _refused(L.mtp_route_topk(3, ONE, 4, 8, 8, 2, 0, ONE, ONE, None, None), b"unknown type")
    _refused(L.mtp_route_topk(0, None, 4, 8, 8, 2, 0, ONE, ONE, None, None), b"null")
    _refused(L.mtp_route_topk_grad(0, ONE, 4, 8, 8, 2, 0, ONE, ONE, None, ONE, ONE, None), b"null")
    _refused(L.mtp_sort_pairs(ONE, -1, 8, ONE, ONE, ONE, None, 0, None), b"bad shape")
    _refused(L.mtp_sort_pairs(ONE, 1 << 31, 8, ONE, ONE, ONE, None, 0, None), b"bad shape")
    _refused(L.mtp_sort_pairs(ONE, 4, 4097, ONE, ONE, ONE, None, 0, None), b"bad shape")
    _refused(L.mtp_sort_pairs(None, 4, 8, ONE, ONE, ONE, None, 0, None), b"null")
    _refused(L.mtp_dispatch_rows(0, ONE, 1 << 30, 8, 8, 4, ONE, ONE, ONE, None), b"bad shape")
    _refused(L.mtp_dispatch_rows(0, ONE, 4, 8, 7, 4, ONE, ONE, ONE, None), b"row distance")
    _refused(L.mtp_combine_rows(0, ONE, 4, 8, 0, ONE, ONE, None, ONE, None), b"bad shape")
    _refused(L.mtp_combine_rows_grad(0, ONE, ONE, 4, 8, 2, ONE, ONE, ONE, None, None, None), b"null")
    _refused(L.mtp_linear(0, ONE, 4, 0, 8, ONE, 8, None, 0, None, 0, None, 1, ONE, None, None, 0, None), b"bad shape")
    _refused(L.mtp_linear(0, ONE, 4, 8, 7, ONE, 8, None, 0, None, 0, None, 1, ONE, None, None, 0, None), b"row distance")
    _refused(L.mtp_linear(0, ONE, 4, 8, 8, ONE, 8, None, 4, None, 0, None, 1, ONE, None, None, 0, None), b"activation")
    _refused(L.mtp_linear(0, ONE, 4, 8, 8, ONE, 8, None, 0, None, 0, None, 2, ONE, None, None, 0, None), b"number of sets")
    _refused(L.mtp_linear(0, ONE, 4, 8, 8, None, 8, None, 0, None, 0, None, 1, ONE, None, None, 0, None), b"null")
    _refused(L.mtp_linear_grad_input(0, ONE, 4, 8, 7, ONE, 8, None, 1, ONE, None, 0, None), b"row distance")
    _refused(L.mtp_linear_grad_weight(0, ONE, 4, 8, 8, None, 8, 8, None, 1, ONE, None, None, 0, None), b"null")
    _refused(L.mtp_linear_act_grad(0, ONE, ONE, 4, 8, 9, None, 1, ONE, 8, None), b"activation")
    _refused(L.mtp_linear_mask_rows(0, ONE, 4, 8, None, 1, ONE, None), b"null")


def test_entry_points_refuse_a_small_workspace():
    L = _lib.lib()
    need = L.mtp_sort_pairs_workspace_bytes(100000, 200)
    assert need > 0 and L.mtp_sort_pairs_workspace_bytes(64, 200) == 0
    assert L.mtp_sort_pairs(ONE, 100000, 200, ONE, ONE, ONE, ONE, need - 1, None) == -3
    assert L.mtp_sort_pairs(ONE, 100000, 200, ONE, ONE, ONE, None, need, None) == -3
    # float rows always start on 4 bytes; a 16-bit row of odd length does not
    assert L.mtp_linear_workspace_bytes(0, _lib.LINEAR_FORWARD, 600, 97, 40, 1, ONE, 97, ONE, 97) == 0
    need = L.mtp_linear_workspace_bytes(1, _lib.LINEAR_FORWARD, 600, 97, 40, 1, ONE, 97, ONE, 97)
    assert need >= (600 + 40) * 104 * 2
    assert L.mtp_linear(1, ONE, 600, 97, 97, ONE, 40, None, 0, None, 0, None, 1, ONE, None, ONE, need - 1, None) == -3
    assert L.mtp_linear(1, ONE, 600, 97, 97, ONE, 40, None, 0, None, 0, None, 1, ONE, None, ONE + 8, need, None) == -3
    # without rows the weights are not read, so they are not laid out anew either
    assert L.mtp_linear_backward_workspace_bytes(1, 0, 97, 41, 1, 0, None, None, 97, None, 97, 1, 1) == 0
    assert L.mtp_linear_backward_workspace_bytes(1, 4, 97, 41, 1, 0, ONE, ONE, 97, ONE, 97, 1, 0) > 0
    need = L.mtp_linear_workspace_bytes(1, _lib.LINEAR_GRAD_WEIGHT, 50000, 96, 40, 1, ONE, 40, ONE, 96)
    assert need > 0 and L.mtp_linear_grad_weight(1, ONE, 50000, 40, 40, ONE, 96, 96, None, 1, ONE, None, ONE, need - 1, None) == -3


def test_nothing_to_do_launches_nothing():
    L = _lib.lib()
    assert L.mtp_route_topk(0, None, 0, 8, 8, 2, 0, None, None, None, None) == 0
    assert L.mtp_linear(0, None, 0, 8, 8, None, 8, None, 0, None, 0, None, 1, None, None, None, 0, None) == 0
    assert L.mtp_combine_rows(0, None, 0, 8, 2, None, None, None, None, None) == 0


def test_front_ends_refuse_cpu_tensors_and_other_things():
    x, ids = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32)
    for call in (lambda: route_topk(x, 2), lambda: sort_pairs(ids, 3), lambda: linear(x, torch.zeros(3, 8)),
                 lambda: modality_linear(x, torch.zeros(3, dtype=torch.int32), torch.zeros(2, 3, 8)),
                 lambda: route_topk(x.requires_grad_(), 2)):
        with pytest.raises(_lib.MtpError):
            call()
    plan = (torch.zeros(3, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), ids)
    from pccs_accel.routing import PairPlan
    for call in (lambda: dispatch(x.detach(), PairPlan(*plan)), lambda: combine(torch.zeros(8, 5), PairPlan(*plan))):
        with pytest.raises(_lib.MtpError):
            call()
    for call in (lambda: route_topk([1.0], 1), lambda: sort_pairs([1], 1), lambda: linear([1.0], x)):
        with pytest.raises(TypeError):
            call()
    with pytest.raises(ValueError):
        K._act_code("tanh")


@pytest.mark.parametrize("kind", [None, "relu", "gelu", "silu"])
def test_formulas_agree_with_autograd(kind):
    g = torch.Generator().manual_seed(0)
    x, w, b, r, gy = (torch.randn(s, generator=g, dtype=torch.float64) for s in ((7, 5), (4, 5), (4,), (7, 4), (7, 4)))
    leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
    z = torch.nn.functional.linear(*leaves[:3])
    y = {None: lambda v: v, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[kind](z) + leaves[3]
    grads = torch.autograd.grad(y, leaves, gy)
    want = R.linear(x, w, b, kind, r, gy)
    for name, v in zip(("y", "dx", "dw", "db", "dres"), (y.detach(),) + grads):
        assert torch.allclose(want[name][0], v, rtol=1e-12, atol=1e-12), name


@pytest.mark.parametrize("normalize", [False, True])
def test_route_formula_agrees_with_autograd(normalize):
    g = torch.Generator().manual_seed(0)
    s = torch.randn(6, 11, generator=g, dtype=torch.float64).requires_grad_()
    gw = torch.randn(6, 3, generator=g, dtype=torch.float64)
    top, ids = torch.topk(s, 3, dim=1)
    w = torch.softmax(top, 1) if normalize else torch.softmax(s, 1).gather(1, ids)
    ds, = torch.autograd.grad(w, s, gw)
    want = R.route(s.detach(), 3, normalize, gw)
    assert torch.equal(want["ids"].long(), ids)
    assert torch.allclose(want["w"][0], w.detach(), rtol=1e-12) and torch.allclose(want["ds"][0], ds, atol=1e-12)


def test_row_distance_of_views():
    t = torch.zeros(6, 10)
    assert K._row_distance(t, "t") == 10 and K._row_distance(t[:, 2:5], "t") == 10 and K._row_distance(t[::2], "t") == 20
    assert K._row_distance(t[:1], "t") == 10 and K._row_distance(t[:, :1], "t") == 10 and K._row_distance(t[:0], "t") == 10
    for bad in (t.T, t[:1].expand(4, 10), t[:, ::2]):
        with pytest.raises(ValueError):
            K._row_distance(bad, "t")
    assert math.isfinite(R.half_step(torch.bfloat16)) and R.half_step(torch.bfloat16) == 2.0 ** -8
