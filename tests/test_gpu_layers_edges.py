"""``pccs_accel.layers`` where a call can go wrong: sums that cancel, saved tensors that come back changed, results that grow."""
import pytest
import torch

import routing_reference as R
from pccs_accel.layers import linear, modality_linear

pytestmark = pytest.mark.gpu


def _bias_gradient_case(rows, out, dtype):
    """One input feature of 1 and 1/2 in turn and weights k / 16: the pre-activations w and w / 2 are exact in every type.  The
    gradient is +1 and -1 in turn, so that the bias' gradient is a small difference of large sums."""
    g = torch.Generator().manual_seed(rows + out)
    w = (torch.randint(-64, 65, (out, 1), generator=g) / 16).to(dtype)
    x = torch.where(torch.arange(rows) % 2 == 0, 1.0, 0.5)[:, None].to(dtype)
    gy = torch.where(torch.arange(rows) % 2 == 0, 1.0, -1.0)[:, None].expand(rows, out).to(dtype).contiguous()
    return x, w, gy


def _bias_gradient(x, w, gy, act):
    """(value, bound): each slope off by 8 roundings of 1 + |z|, a float32 sum of as many terms as rows, one rounding to the type."""
    z = x.double() @ w.double().T
    dz = gy.double() * R.slope(z, act)
    v = dz.sum(0)
    e = (8 * R.U32 * (1 + z.abs())).sum(0) + (x.shape[0] + 2) * R.U32 * dz.abs().sum(0)
    return v, e + R.half_step(x.dtype) * (v.abs() + e) + R.floor_of(x.dtype)


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("size", [(1, 3), (2, 1), (16, 8), (17, 201), (300, 9), (333, 2048), (1001, 2057), (5000, 64), (20000, 7)], ids=str)
def test_bias_gradient_is_a_sum_of_what_is_not_rounded(gpu_device, size, act):
    for dtype in R.TYPES:
        x, w, gy = _bias_gradient_case(*size, dtype)
        bias = torch.zeros(size[1], dtype=dtype, device=gpu_device).requires_grad_()
        db, = torch.autograd.grad(linear(x.to(gpu_device), w.to(gpu_device), bias, act), bias, gy.to(gpu_device))
        assert db.dtype == dtype
        R.check("db", db, _bias_gradient(x, w, gy, act))


@pytest.mark.parametrize("sets,size", [(3, (100, 40)), (7, (3000, 201)), (600, (2500, 24)), (40, (9000, 256))], ids=str)
def test_bias_gradients_of_modalities_are_sums_of_what_is_not_rounded(gpu_device, sets, size):
    """Empty modalities, one that has most rows, and rows behind the last one whose gradient is NaN."""
    rows, out = size
    g = torch.Generator().manual_seed(sets)
    who = torch.where(torch.rand(rows - 5, generator=g) < 0.5, torch.full((rows - 5,), sets // 2), torch.randint(0, sets - 1, (rows - 5,), generator=g))
    offsets = torch.cat([torch.zeros(1).long(), torch.bincount(who, minlength=sets).cumsum(0)]).to(torch.int32)
    for dtype in (torch.bfloat16, torch.float16):
        x, _, gy = _bias_gradient_case(rows, out, dtype)
        gy[rows - 5:] = float("nan")
        w = (torch.randint(-64, 65, (sets, out, 1), generator=g) / 16).to(dtype)
        bias = torch.zeros(sets, out, dtype=dtype, device=gpu_device).requires_grad_()
        y = modality_linear(x.to(gpu_device), offsets.to(gpu_device), w.to(gpu_device), bias, "gelu")
        db, = torch.autograd.grad(y, bias, gy.to(gpu_device))
        at = offsets.tolist()
        want = [_bias_gradient(x[at[e]:at[e + 1]], w[e], gy[at[e]:at[e + 1]], "gelu") for e in range(sets)]
        R.check("db", db, (torch.stack([v for v, _ in want]), torch.stack([e for _, e in want])))
