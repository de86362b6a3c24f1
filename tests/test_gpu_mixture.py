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


def _expected(net, obs, labels, mods):
    """Displacements of the agents' candidates ``labels`` [N, k], and how far two evaluations in the net's type may be apart: the
    synthesizer's and the decoder's results are rounded once each, on either side."""
    n, k = labels.shape
    many = obs.repeat_interleave(k, dim=0)
    future = net.synthesizer(many, labels=labels.reshape(-1), all_modalities=mods)
    out = net.decoder([many, future])
    size = torch.cat((many, future), 1).double().abs() @ net.decoder.fc.weight.double().abs().T + net.decoder.fc.bias.double().abs()
    return (v.reshape(n, k, T, 2).cpu().double() for v in (out, 4 * R.half_step(obs.dtype) * 0.25 * size))


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
@pytest.mark.parametrize("normalize", [True, False])
def test_candidates_and_weights_go_by_the_probabilities_themselves(gpu_device, dtype, normalize):
    """Neighbouring 16-bit probabilities have the same logarithm in their type: order and weights come from the former."""
    net = _net(dtype).to(gpu_device)
    obs, mods = (t.to(gpu_device) for t in _inputs(dtype))
    for k in (1, 5, 12):
        with torch.no_grad():
            disp, weights, mean = predict_mixture(net, obs, k, mods, normalize=normalize)
            top = torch.sort(net.classifier(obs).cpu(), dim=1, descending=True, stable=True)
            labels = top.indices[:, :k]
            want, bound = _expected(net, obs, labels.to(gpu_device), mods)
        assert weights.dtype == torch.float32 and disp.dtype == dtype
        w = top.values[:, :k].double()
        w = w / w.sum(1, keepdim=True) if normalize else w
        R.check("weights", weights, (w, (k + 4) * R.U32 * w))
        R.check("displacements", disp, (want, bound))
        exact = (w[:, :, None, None] * disp.cpu().double()).sum(1)
        size = (w[:, :, None, None] * disp.cpu().double().abs()).sum(1)
        R.check("mean", mean, (exact, (2 * k + 8) * R.U32 * size + R.half_step(dtype) * (exact.abs() + size * 1e-4) + R.floor_of(dtype)))


def test_candidates_of_probability_zero_are_the_agents_own(gpu_device):
    """Three probabilities are not zero and six candidates wanted: the others are the lowest modalities, for this agent, with weight 0."""
    for dtype in R.TYPES:
        net = _net(dtype, all_but=(2, 3, 9)).to(gpu_device)
        obs, mods = (t.to(gpu_device) for t in _inputs(dtype))
        with torch.no_grad():
            disp, weights, mean = predict_mixture(net, obs, 6, mods)
            top = torch.sort(net.classifier(obs).cpu(), dim=1, descending=True, stable=True).indices[:, :6]
            want, bound = _expected(net, obs, top.to(gpu_device), mods)
        assert (top[:, 3:] == torch.tensor([0, 1, 4])).all() and (weights[:, 3:] == 0).all()
        R.check("displacements", disp, (want, bound))
        assert torch.isfinite(mean).all()


def test_a_probability_that_is_nan_makes_its_agents_weights_nan(gpu_device):
    net = _net(torch.float32).to(gpu_device)
    obs, mods = (t.to(gpu_device) for t in _inputs(torch.float32))
    obs[4, 0] = float("nan")
    with torch.no_grad():
        disp, weights, mean = predict_mixture(net, obs, 5, mods)
    keep = [i for i in range(N) if i != 4]
    assert torch.isnan(weights[4]).all()
    assert torch.isfinite(weights[keep]).all() and torch.isfinite(mean[keep]).all() and torch.isfinite(disp[keep]).all()
