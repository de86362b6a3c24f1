"""Calls of the routing and layer operators that are refused before they look at a device: these run without one."""
import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

from pccs_accel.layers import linear, modality_linear
from pccs_accel.routing import PairPlan, combine, dispatch, route_topk, sort_pairs


def _calls():
    x, w, ids = torch.randn(4, 8), torch.randn(3, 8), torch.zeros(4, 2, dtype=torch.int32)
    plan = PairPlan(torch.zeros(4, dtype=torch.int32), torch.zeros(8, dtype=torch.int32), ids)
    rows, w3 = torch.randn(8, 5), torch.randn(3, 6, 8)
    return [(lambda t: route_topk(t, 2), x), (lambda t: sort_pairs(t, 3), ids), (lambda t: dispatch(t, plan), x),
            (lambda t: combine(t, plan), rows), (lambda t: linear(t, w), x), (lambda t: modality_linear(t, plan.offsets, w3), x)]


@pytest.mark.parametrize("which", range(6))
def test_tracing_is_refused(which):
    """A trace would hold uninitialised memory, or the values of the traced call, in place of the results."""
    call, given = _calls()[which]
    with pytest.raises(RuntimeError, match="cannot be traced"):
        torch.jit.trace(call, (given,), check_trace=False)
    for mode in ("real", "fake"):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            make_fx(call, tracing_mode=mode)(given)
