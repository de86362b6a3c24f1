"""The routing and layer operators at the ends of what they accept: one modality with many rows, the longest rows and sums, the widest
row distances."""
import pytest
import torch

import routing_reference as R
from pccs_accel.layers import linear, modality_linear
from pccs_accel.routing import combine, dispatch, sort_pairs

pytestmark = pytest.mark.gpu


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def _check_layer(dev, x, w, b, act, gy, offsets=None, on_device=None):
    leaves = [(on_device if on_device is not None else x.to(dev)).requires_grad_(), w.to(dev).requires_grad_(), b.to(dev).requires_grad_()]
    if offsets is None:
        y, want = linear(*leaves, activation=act), R.linear(x, w, b, act, None, gy)
    else:
        y, want = modality_linear(leaves[0], offsets.to(dev), *leaves[1:], activation=act), R.modality_linear(x, offsets, w, b, act, None, gy)
    grads = torch.autograd.grad(y, leaves, gy.to(dev))
    for name, v in zip(("y", "dx", "dw", "db"), (y,) + grads):
        R.check(name, v, want[name])


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
@pytest.mark.parametrize("size", [(9000, 600, 520, 100), (700, 40, 24, 0), (20000, 33, 129, 1)], ids=str)
def test_one_modality_has_all_rows(gpu_device, size, dtype):
    rows, i, o, behind = size
    g = torch.Generator().manual_seed(rows)
    x, w, b, gy = _normal(g, (rows, i), dtype), _normal(g, (1, o, i), dtype, i ** -0.5), _normal(g, (1, o), dtype), _normal(g, (rows, o), dtype)
    _check_layer(gpu_device, x, w, b, "gelu", gy, torch.tensor([0, rows - behind], dtype=torch.int32))


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
@pytest.mark.parametrize("size", [(5, 65536, 3), (600, 65536, 2), (3, 2, 65536), (600, 3, 65535)], ids=str)
def test_longest_sums_and_widest_results(gpu_device, size, dtype):
    rows, i, o = size
    g = torch.Generator().manual_seed(i + o)
    x, w, b, gy = _normal(g, (rows, i), dtype), _normal(g, (o, i), dtype, i ** -0.5), _normal(g, (o,), dtype), _normal(g, (rows, o), dtype)
    _check_layer(gpu_device, x, w, b, "silu", gy)


@pytest.mark.parametrize("rows", [20, 600])
def test_rows_far_apart(gpu_device, rows):
    """A slice of columns of a matrix whose rows are more than 2^20 elements long."""
    g = torch.Generator().manual_seed(rows)
    for dtype in (torch.float32, torch.float16):
        whole = torch.zeros(rows, (1 << 20) + 7, dtype=dtype, device=gpu_device)
        x = _normal(g, (rows, 50), dtype)
        whole[:, 3:53] = x.to(gpu_device)
        w, b, gy = _normal(g, (30, 50), dtype, 0.1), _normal(g, (30,), dtype), _normal(g, (rows, 30), dtype)
        _check_layer(gpu_device, x, w, b, "gelu", gy, on_device=whole[:, 3:53])
        plan = sort_pairs(torch.randint(0, 5, (rows, 2), generator=g, dtype=torch.int32).to(gpu_device), 5)
        assert torch.equal(dispatch(whole[:, 3:53], plan), dispatch(x.to(gpu_device), plan))


@pytest.mark.parametrize("d", [1 << 20, (1 << 20) - 3])
def test_longest_rows_there_and_back(gpu_device, d):
    g = torch.Generator().manual_seed(d)
    plan = sort_pairs(torch.tensor([[0, 2], [1, -1], [2, 0]], dtype=torch.int32).to(gpu_device), 3)
    there = torch.tensor([[1.0, 1.0], [1.0, 0.0], [1.0, 1.0]], dtype=torch.float64)
    here = plan.position.cpu().long()
    for dtype in (torch.float32, torch.bfloat16):
        u = R.half_step(dtype)
        x, rows, gy, w = _normal(g, (3, d), dtype), _normal(g, (6, d), dtype), _normal(g, (3, d), dtype), torch.rand(3, 2, generator=g)
        out = dispatch(x.to(gpu_device), plan).cpu()
        assert torch.equal(out[here.reshape(-1)], (x[:, None].double() * there[:, :, None]).reshape(6, d).to(dtype))
        leaves = rows.to(gpu_device).requires_grad_(), w.to(gpu_device).requires_grad_()
        y = combine(leaves[0], plan, leaves[1])
        terms = rows.double()[here] * (w.double() * there)[:, :, None]
        v, e = terms.sum(1), 4 * R.U32 * terms.abs().sum(1)
        R.check("y", y, (v, e + u * (v.abs() + e) + R.floor_of(dtype)))
        dr, dw = torch.autograd.grad(y, leaves, gy.to(gpu_device))
        back = (w.double() * there)[:, :, None] * gy.double()[:, None]
        R.check("drows", dr[plan.position.long()], (back, (u + 2 * R.U32) * back.abs() + R.floor_of(dtype)))
        prod = rows.double()[here] * gy.double()[:, None] * there[:, :, None]
        R.check("dw", dw, (prod.sum(2), (d + 2) * R.U32 * prod.abs().sum(2)))
    with pytest.raises(RuntimeError, match="bad shape"):
        dispatch(torch.zeros(3, (1 << 20) + 1, device=gpu_device), plan)
