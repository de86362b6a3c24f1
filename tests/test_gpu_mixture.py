"""``evaluation.predict_mixture`` where probabilities vanish and where they are 16 bits wide, against the formulas in float64."""
import pytest
import torch

import routing_reference as R
from pccs_accel.evaluation import predict_mixture
from test_gpu_glue import _ToyNet

pytestmark = pytest.mark.gpu

N, F, C, T = 23, 16, 12, 12


def _net(dtype, gone=(), all_but=None):
    """The toy net with logits so low that the modalities ``gone`` have probability zero (``all_but``: all but these)."""
    net = _ToyNet(F, C, T)
    gone = [c for c in range(C) if c not in all_but] if all_but is not None else list(gone)
    with torch.no_grad():
        net.classifier.fc.bias[gone] = -300.0
    return net.to(dtype)


def _inputs(dtype, seed=3):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(N, F, generator=g).to(dtype), torch.randn(C, 2 * F, generator=g).to(dtype)


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("k,gone", [(4, (0, 7)), (12, (0, 7)), (8, (0, 1, 2, 3, 4, 6)), (1, (5,))], ids=str)
def test_gradients_are_finite_where_probabilities_are_zero(gpu_device, k, gone, normalize):
    """Modalities of probability zero among the k and outside them."""
    net = _net(torch.float32, gone).to(gpu_device)
    obs, mods = _inputs(torch.float32)
    leaf = obs.to(gpu_device).requires_grad_()
    params = [leaf] + list(net.parameters())
    _, weights, mean = predict_mixture(net, leaf, k, mods.to(gpu_device), normalize=normalize)
    assert torch.isfinite(weights).all() and (net.classifier(leaf)[:, list(gone)] == 0).all()
    got = torch.autograd.grad(mean.square().sum() + (weights * weights).sum(), params)
    ref = _net(torch.float64, gone)
    leaf64 = obs.double().requires_grad_()
    probs = ref.classifier(leaf64)
    top = torch.sort(probs, dim=1, descending=True, stable=True)
    w = top.values[:, :k] / (top.values[:, :k].sum(1, keepdim=True) if normalize else 1)
    many = leaf64.repeat_interleave(k, dim=0)
    out = ref.decoder([many, ref.synthesizer(many, labels=top.indices[:, :k].reshape(-1), all_modalities=mods.double())])
    mean64 = (w[:, :, None, None] * out.reshape(N, k, T, 2)).sum(1)
    want = torch.autograd.grad(mean64.square().sum() + (w * w).sum(), [leaf64] + list(ref.parameters()))
    for a, c in zip(got, want):  # float32 sums of at most N k terms of up to 2 F products each
        a = a.cpu().double()
        assert torch.isfinite(a).all() and float((a - c).norm()) <= N * k * 2 * F * R.U32 * float(c.norm()) + 1e-12
