"""``pccs_accel.routing`` on the GPU against float64 formulas (routing_reference.py), and the routed layers as they run together."""
import io
import math

import pytest
import torch

import routing_reference as R
from pccs_accel import kernels as K
from pccs_accel.layers import modality_linear
from pccs_accel.routing import PairPlan, combine, dispatch, route_topk, sort_pairs

pytestmark = pytest.mark.gpu

# rows, modalities, k: one agent, every width of the kernel (64, 256, 512, 1024, 4096), few and many rows, k up to all
ROUTES = [(1, 1, 1), (1, 200, 20), (3, 7, 7), (5, 64, 1), (1030, 5, 3), (1500, 64, 64), (1025, 65, 17), (1200, 200, 20), (900, 256, 128),
          (1100, 257, 33), (1050, 400, 7), (1040, 1024, 128), (30, 1024, 8), (7, 1025, 5), (2, 4096, 128), (1024, 33, 32), (1026, 999, 16),
          (1030, 130, 4), (1040, 300, 8), (1050, 511, 9), (1060, 512, 20), (1030, 513, 70), (1100, 8, 8), (1100, 9, 9)]
# eight lanes a row: every width and batch of choices, their borders, rows that end inside a piece
ROUTES += [(1024, 1, 1), (1031, 7, 2), (1024, 31, 31), (1057, 32, 9), (1033, 40, 17), (1039, 64, 33), (1025, 100, 8), (1041, 127, 100),
           (1029, 128, 128), (1030, 129, 33), (1037, 201, 70), (1026, 256, 128), (1027, 256, 32)]


def _scores(seed, n, e, dtype):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(n, e, generator=g) * 2).to(dtype)


def _route(dev, scores, k, normalize, g):
    leaf = scores.to(dev).requires_grad_()
    ids, w = route_topk(leaf, k, normalize=normalize)
    assert ids.dtype == torch.int32 and w.dtype == torch.float32
    ds, = torch.autograd.grad(w, leaf, g.to(dev))
    plain_ids, plain_w = route_topk(scores.to(dev), k, normalize=normalize)
    assert torch.equal(plain_ids, ids) and torch.equal(plain_w.nan_to_num(7), w.detach().nan_to_num(7))
    return ids, w, ds


def _check_route(dev, scores, k, normalize, seed=0):
    g = torch.randn(scores.shape[0], k, generator=torch.Generator().manual_seed(seed))
    want = R.route(scores, k, normalize, g)
    ids, w, ds = _route(dev, scores, k, normalize, g)
    assert torch.equal(ids.cpu(), want["ids"])
    R.check("w", w, want["w"])
    assert ds.dtype == scores.dtype
    R.check("ds", ds, want["ds"])


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
@pytest.mark.parametrize("size", ROUTES, ids=str)
def test_route_and_gradient(gpu_device, size, dtype):
    n, e, k = size
    for normalize in (False, True):
        _check_route(gpu_device, _scores(n + e, n, e, dtype), k, normalize)


@pytest.mark.parametrize("n", [3, 1100])
def test_route_ties_go_to_the_lowest_index(gpu_device, n):
    for dtype in R.TYPES:
        g = torch.Generator().manual_seed(1)
        scores = torch.randint(-2, 3, (n, 150), generator=g).to(dtype)
        scores[0] = 0
        scores[1, ::2] = -0.0  # equals +0
        scores[1, 1::2] = 0.0
        _check_route(gpu_device, scores, 40, True)
        _check_route(gpu_device, scores, 40, False)


@pytest.mark.parametrize("e,k", [(20, 12), (50, 30), (110, 50), (250, 60)])
def test_route_eight_lanes_masks_and_ties(gpu_device, e, k):
    """Rows with fewer than k scores left, rows of equal scores, NaN: lanes run out of keys at different times."""
    for dtype in R.TYPES:
        scores = _scores(e, 1033, e, dtype)
        scores[0] = -math.inf
        scores[1, 3:] = -math.inf
        scores[2] = 1.0
        scores[3] = torch.arange(e).to(dtype)          # the best in the last lanes
        scores[4] = -torch.arange(e).to(dtype)         # and in the first
        scores[5, ::3] = -math.inf
        scores[1032, 1:] = -math.inf                   # the last row, which fills the rest of its workgroup
        for normalize in (False, True):
            _check_route(gpu_device, scores, k, normalize)
        scores[6, e // 2] = math.nan
        ids, w = route_topk(scores.to(gpu_device), k)
        assert torch.isnan(w[6]).all() and not torch.isnan(w[5]).any() and not torch.isnan(w[7]).any()
        assert int(ids[6].max()) < e


@pytest.mark.parametrize("n", [6, 1200])
def test_route_masked_rows(gpu_device, n):
    for dtype in R.TYPES:
        for normalize in (False, True):
            scores = _scores(3, n, 90, dtype)
            scores[0] = -math.inf                     # nothing allowed
            scores[1, 5:] = -math.inf                 # fewer than k
            scores[2] = torch.finfo(dtype).min        # lowest value: allowed, and a tie
            scores[3, :] = -math.inf
            scores[3, 77] = torch.finfo(dtype).max
            _check_route(gpu_device, scores, 9, normalize)
            ids, w = route_topk(scores.to(gpu_device), 9, normalize=normalize)
            assert (ids[0] == -1).all() and (w[0] == 0).all() and (ids[1, 5:] == -1).all()
            assert ids[3].tolist() == [77] + [-1] * 8 and w[3, 0] == 1


def test_route_nan_and_infinity(gpu_device):
    for n in (4, 1100):
        for normalize in (False, True):
            scores = _scores(4, n, 70, torch.float32)
            scores[1, 3] = math.nan
            scores[2, 8] = math.inf
            ids, w = route_topk(scores.to(gpu_device), 70, normalize=normalize)
            assert torch.isnan(w[1]).all() and 3 not in ids[1, :69].tolist() and ids[1, 69] == -1
            assert ids[2, 0] == 8 and torch.isnan(w[2, 0])
            keep = [0, 3]
            assert torch.isfinite(w[keep]).all()


def test_route_large_scores_keep_their_precision(gpu_device):
    """Differences count, not sizes: scores around 30 000 in float32."""
    scores = _scores(5, 40, 60, torch.float32) + 30000.0
    for normalize in (False, True):
        _check_route(gpu_device, scores, 12, normalize)


def test_route_takes_a_slice_of_columns(gpu_device):
    for dtype in R.TYPES:
        wide = _scores(6, 1100, 131, dtype)
        want = R.route(wide[:, 7:97], 5, True)
        ids, w = route_topk(wide.to(gpu_device)[:, 7:97], 5)
        assert torch.equal(ids.cpu(), want["ids"])
        R.check("w", w, want["w"])


def test_route_gradient_against_differences(gpu_device):
    scores = _scores(8, 6, 30, torch.float32)
    g = torch.randn(6, 4, generator=torch.Generator().manual_seed(2))
    for normalize in (False, True):
        ids, w, ds = _route(gpu_device, scores, 4, normalize, g)
        ids = ids.cpu().long()
        d = torch.randn(6, 30, generator=torch.Generator().manual_seed(3), dtype=torch.float64)

        def value(h):
            s = scores.double() + h * d
            top = s.gather(1, ids)
            return float((g.double() * torch.exp(top - torch.logsumexp(top if normalize else s, 1, keepdim=True))).sum())
        slope = (value(1e-4) - value(-1e-4)) / 2e-4
        err = float((R.route(scores, 4, normalize, g)["ds"][1] * d.abs()).sum())
        # central differences: h^2 / 6 times the third derivative of a softmax along d (at most some 6 max|d|^3 sum|g|)
        err += 1e-8 * float(d.abs().max()) ** 3 * float(g.abs().sum()) + 1e-10
        assert abs(float((ds.cpu().double() * d).sum()) - slope) <= err


PAIRS = [(0, 3, 5), (1, 1, 1), (1, 20, 200), (5, 3, 2), (63, 1, 4), (64, 1, 4), (65, 2, 7), (1000, 4, 300), (3000, 5, 200), (900, 8, 4096),
         (5000, 4, 1), (17970, 4, 400), (40000, 3, 1024), (9000, 2, 4096)]


@pytest.mark.parametrize("size", PAIRS, ids=str)
def test_sort_pairs(gpu_device, size):
    n, k, e = size
    g = torch.Generator().manual_seed(n + e)
    for low in (0, -1):
        ids = torch.randint(low, e, (n, k), generator=g, dtype=torch.int32)
        if low < 0 and n:
            ids[n // 2] = e + 3  # out of range counts as none
        key = ids.reshape(-1).long()
        key = torch.where((key < 0) | (key >= e), torch.full_like(key, e), key)
        order = torch.sort(key, stable=True).indices
        position = torch.empty_like(order)
        position[order] = torch.arange(n * k)
        plan = sort_pairs(ids.to(gpu_device), e)
        offsets = torch.cat([torch.zeros(1).long(), torch.bincount(key, minlength=e + 1)[:e].cumsum(0)])
        assert torch.equal(plan.offsets.cpu().long(), offsets)
        assert torch.equal(plan.order.cpu().long(), order)
        assert torch.equal(plan.position.cpu().long(), position.view(n, k))


def _plan(seed, n, k, e, none=0.0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, e, (n, k), generator=g, dtype=torch.int32)
    ids[torch.rand(n, k, generator=g) < none] = -1
    return ids


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
@pytest.mark.parametrize("size", [(1, 1, 1, 3), (1, 20, 96, 200), (7, 3, 33, 5), (50, 2, 8, 4), (129, 4, 96, 30), (40, 5, 130, 9),
                                  (700, 20, 48, 200), (33, 2, 1024, 6), (2000, 1, 64, 50), (3, 4, 520, 7)], ids=str)
def test_rows_there_and_back(gpu_device, size, dtype):
    n, k, d, e = size
    u = R.half_step(dtype)
    for none in (0.0, 0.3):
        ids = _plan(n + d, n, k, e, none)
        plan = sort_pairs(ids.to(gpu_device), e)
        g = torch.Generator().manual_seed(d)
        x = torch.randn(n, d, generator=g).to(dtype)
        rows = torch.randn(n * k, d, generator=g).to(dtype)
        w = torch.rand(n, k, generator=g)
        g_rows, g_y = torch.randn(n * k, d, generator=g).to(dtype), torch.randn(n, d, generator=g).to(dtype)
        here = plan.position.cpu().long()
        there = ((ids >= 0) & (ids < e)).double()

        xd = x.to(gpu_device).requires_grad_()
        out = dispatch(xd, plan)
        want = torch.zeros(n * k, d, dtype=dtype)
        want[here.reshape(-1)] = (x.double()[:, None, :] * there[:, :, None]).reshape(-1, d).to(dtype)
        assert torch.equal(out.cpu(), want)
        dx, = torch.autograd.grad(out, xd, g_rows.to(gpu_device))
        terms = g_rows.double()[here] * there[:, :, None]
        v, e32 = terms.sum(1), (k + 2) * R.U32 * terms.abs().sum(1)
        R.check("dx", dx, (v, e32 + u * (v.abs() + e32) + R.floor_of(dtype)))

        rd, wd = rows.to(gpu_device).requires_grad_(), w.to(gpu_device).requires_grad_()
        y = combine(rd, plan, wd)
        terms = rows.double()[here] * (w.double() * there)[:, :, None]
        v, e32 = terms.sum(1), (k + 2) * R.U32 * terms.abs().sum(1)
        R.check("y", y, (v, e32 + u * (v.abs() + e32) + R.floor_of(dtype)))
        dr, dw = torch.autograd.grad(y, [rd, wd], g_y.to(gpu_device))
        back = torch.zeros(n * k, d, dtype=torch.float64)
        back[here.reshape(-1)] = ((w.double() * there)[:, :, None] * g_y.double()[:, None, :]).reshape(-1, d)
        R.check("drows", dr, (back, (u + 2 * R.U32) * back.abs() + R.floor_of(dtype)))
        prod = rows.double()[here] * g_y.double()[:, None, :] * there[:, :, None]
        R.check("dw", dw, (prod.sum(2), (d + 2) * R.U32 * prod.abs().sum(2)))

        rd = rows.to(gpu_device).requires_grad_()
        y = combine(rd, plan)
        terms = rows.double()[here] * there[:, :, None]
        v, e32 = terms.sum(1), (k + 2) * R.U32 * terms.abs().sum(1)
        R.check("sum", y, (v, e32 + u * (v.abs() + e32) + R.floor_of(dtype)))
        dr, = torch.autograd.grad(y, rd, g_y.to(gpu_device))
        back = torch.zeros(n * k, d, dtype=dtype)
        back[here.reshape(-1)] = (g_y.double()[:, None, :] * there[:, :, None]).reshape(-1, d).to(dtype)
        assert torch.equal(dr.cpu(), back)


def test_rows_from_a_slice_and_without_agents(gpu_device):
    plan = sort_pairs(_plan(1, 40, 3, 6).to(gpu_device), 6)
    wide = torch.randn(40, 70, generator=torch.Generator().manual_seed(1)).to(gpu_device)
    for start in (0, 1, 4):
        assert torch.equal(dispatch(wide[:, start:start + 48], plan), dispatch(wide[:, start:start + 48].contiguous(), plan))
    empty = sort_pairs(torch.empty(0, 3, dtype=torch.int32, device=gpu_device), 6)
    assert dispatch(wide[:0], empty).shape == (0, 70) and combine(wide[:0], empty, wide[:0, :3].contiguous()).shape == (0, 70)


def test_rows_that_nobody_answers_may_hold_anything(gpu_device):
    """NaN behind the last modality's rows does not reach a sum or a gradient."""
    ids = _plan(2, 30, 4, 5, none=0.5)
    plan = sort_pairs(ids.to(gpu_device), 5)
    rows = torch.randn(120, 24, generator=torch.Generator().manual_seed(2)).to(gpu_device)
    held = int(plan.offsets[-1])
    clean = combine(rows, plan, torch.ones(30, 4, device=gpu_device))
    rows[held:] = math.nan
    w = torch.ones(30, 4, device=gpu_device, requires_grad=True)
    leaf = rows.clone().requires_grad_()
    y = combine(leaf, plan, w)
    assert torch.equal(y, clean)
    dr, dw = torch.autograd.grad(y, [leaf, w], torch.ones_like(y))
    assert torch.isfinite(dr).all() and torch.isfinite(dw).all() and not dr[held:].any()


def _layer(scores, x, w1, b1, w2, b2, k):
    """Two layers per modality over each agent's k modalities, averaged with the router's weights."""
    ids, w = route_topk(scores, k)
    plan = sort_pairs(ids, scores.shape[1])
    hidden = modality_linear(dispatch(x, plan), plan.offsets, w1, b1, activation="gelu")
    return combine(modality_linear(hidden, plan.offsets, w2, b2), plan, w)


def _layer_inputs(n, e, d, h, o, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, e, generator=g) * 2).to(dtype), torch.tanh(torch.randn(n, d, generator=g)).to(dtype),
            (torch.randn(e, h, d, generator=g) / d ** 0.5).to(dtype), (torch.randn(e, h, generator=g) * 0.1).to(dtype),
            (torch.randn(e, o, h, generator=g) / h ** 0.5).to(dtype), (torch.randn(e, o, generator=g) * 0.1).to(dtype)]


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
@pytest.mark.parametrize("size", [(1, 200, 4, 96, 64, 24), (37, 12, 3, 17, 33, 5), (500, 20, 6, 48, 64, 24)], ids=str)
def test_routed_layers_together(gpu_device, size, dtype):
    n, e, k, d, h, o = size
    inputs = _layer_inputs(n, e, d, h, o, dtype)
    inputs[0][n // 2, 2:] = -math.inf  # an agent with two modalities left
    gy = torch.randn(n, o, generator=torch.Generator().manual_seed(5)).to(dtype)
    exact = [t.double().requires_grad_() for t in inputs]
    s, x, w1, b1, w2, b2 = exact
    ids = R.route(inputs[0], k, True)["ids"].long()
    y = 0
    top = s.gather(1, ids.clamp_min(0)).masked_fill(ids < 0, -math.inf)
    weight = torch.softmax(top, 1)
    for j in range(k):
        e_j = ids[:, j].clamp_min(0)
        hidden = R.act(torch.einsum("nd,nhd->nh", x, w1[e_j]) + b1[e_j], "gelu")
        y = y + (weight[:, j] * (ids[:, j] >= 0))[:, None] * (torch.einsum("nh,noh->no", hidden, w2[e_j]) + b2[e_j])
    want = torch.autograd.grad(y, exact, gy.double())
    leaves = [t.to(gpu_device).requires_grad_() for t in inputs]
    out = _layer(*leaves, k)
    got = torch.autograd.grad(out, leaves, gy.to(gpu_device))
    # each of the (at most ten) tensors between the inputs and a gradient is rounded to the type once, float32 sums of at most
    # n * k terms on the way: 2-norm of the error against the 2-norm of the result, roundings added up, twice over for cancellation
    most = 2 * (10 * R.half_step(dtype) + 4 * (n * k + d + h) * R.U32)
    for name, a, c in zip(("y", "scores", "x", "w1", "b1", "w2", "b2"), (out,) + got, (y,) + want):
        a, c = a.detach().cpu().double(), c.detach()
        assert float((a - c).norm()) <= most * float(c.norm()), (name, float((a - c).norm() / c.norm()), most)


def test_routed_layers_in_graphs_and_streams(gpu_device):
    """Two captured graphs replayed in turn with eager work between, and two streams at once."""
    base = [t.to(gpu_device) for t in _layer_inputs(300, 50, 32, 40, 24, torch.bfloat16)]
    gy = torch.randn(300, 24, generator=torch.Generator().manual_seed(5)).to(gpu_device).to(torch.bfloat16)

    def step(inputs):
        leaves = [t.detach().requires_grad_() for t in inputs]
        y = _layer(*leaves, 5)
        return [y.detach()] + list(torch.autograd.grad(y, leaves, gy))
    side = torch.cuda.Stream()
    graphs = []
    for _ in range(2):
        static = [t.clone() for t in base]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(static)
        graphs.append((graph, static, outs))
    for turn in range(4):
        for graph, static, outs in graphs:
            for t, src in zip(static, base):
                t.copy_(src * (1 - 0.2 * turn))
            graph.replay()
            torch.cuda.synchronize()
            for a, c in zip(outs, step([t.clone() for t in static])):
                assert torch.equal(a, c)
    want = step(base)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(step(base))
    torch.cuda.synchronize()
    for outs in got:
        for a, c in zip(outs, want):
            assert torch.equal(a, c)


def test_refusals(gpu_device):
    d = gpu_device
    s = torch.zeros(4, 9, device=d)
    ids = torch.zeros(4, 2, dtype=torch.int32, device=d)
    plan = sort_pairs(ids, 9)
    for call, error in [
        (lambda: route_topk(s.cpu(), 2), K._lib.MtpError),
        (lambda: route_topk(s.double(), 2), TypeError),
        (lambda: route_topk(s[0], 2), ValueError),
        (lambda: route_topk(s, 0), ValueError),
        (lambda: route_topk(s, 10), ValueError),
        (lambda: route_topk(torch.zeros(2, 300, device=d), 129), ValueError),
        (lambda: route_topk(torch.zeros(2, 4097, device=d), 2), ValueError),
        (lambda: route_topk(s.T, 2), ValueError),
        (lambda: route_topk(s[:1].expand(4, 9), 2), ValueError),
        (lambda: sort_pairs(ids.long(), 9), TypeError),
        (lambda: sort_pairs(ids.cpu(), 9), K._lib.MtpError),
        (lambda: sort_pairs(ids[:, :1], 9), ValueError),
        (lambda: sort_pairs(ids.view(-1), 9), ValueError),
        (lambda: sort_pairs(ids, 0), ValueError),
        (lambda: sort_pairs(ids, 4097), ValueError),
        (lambda: dispatch(s[:3], plan), ValueError),
        (lambda: dispatch(s.long(), plan), TypeError),
        (lambda: combine(s, plan), ValueError),
        (lambda: combine(torch.zeros(8, 9, device=d), plan, torch.zeros(4, 3, device=d)), ValueError),
        (lambda: combine(torch.zeros(8, 9, device=d), plan, torch.zeros(4, 2, device=d).half()), TypeError),
        (lambda: combine(torch.zeros(9, 8, device=d).T, plan), ValueError),
        (lambda: combine(torch.zeros(8, 9, device=d), PairPlan(plan.offsets.long(), plan.order, plan.position)), TypeError),
    ]:
        with pytest.raises(error):
            call()


def test_second_derivatives_are_refused(gpu_device):
    s = _scores(1, 6, 20, torch.float32).to(gpu_device).requires_grad_()
    ids, w = route_topk(s, 3)
    ds, = torch.autograd.grad(w[:, 0].sum(), s, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(ds.square().sum(), s)
    plan = sort_pairs(ids, 20)
    x = torch.randn(6, 8, device=gpu_device, requires_grad=True)
    rows = torch.randn(18, 8, device=gpu_device, requires_grad=True)
    g = torch.randn(18, 8, device=gpu_device, requires_grad=True)
    dx, = torch.autograd.grad(dispatch(x, plan), x, g, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(dx.sum(), g)
    weights = w.detach().requires_grad_()
    dr, dw = torch.autograd.grad(combine(rows, plan, weights).square().sum(), [rows, weights], create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(dr.sum() + dw.sum(), rows)


def test_predict_mixture_is_predict_topk_with_weights(gpu_device):
    """Candidates as predict_topk gives them (the toy net's probabilities differ), weights and mean by their formulas, gradients."""
    from pccs_accel.evaluation import predict_mixture, predict_topk
    from test_gpu_glue import _ToyNet
    net = _ToyNet().to(gpu_device)
    g = torch.Generator().manual_seed(3)
    obs = torch.randn(29, 16, generator=g).to(gpu_device)
    mods = torch.randn(12, 32, generator=g).to(gpu_device)
    for k in (1, 5, 12):
        with torch.no_grad():
            want = predict_topk(net, obs, k, mods)
            disp, weights, mean = predict_mixture(net, obs, k, mods)
            p = net.classifier(obs).double().sort(dim=1, descending=True).values[:, :k]
        # the same float32 products over rows in another order: the library may choose another kernel, 32 terms each
        assert torch.allclose(disp, want, rtol=0, atol=64 * R.U32 * float(want.abs().max()) + 64 * R.U32)
        w = (p / p.sum(1, keepdim=True)).cpu()
        R.check("weights", weights, (w, 128 * R.U32 * w))  # log and exp of probabilities down to e^-30
        exact = (w[:, :, None, None] * disp.cpu().double()).sum(1)
        size = (w[:, :, None, None] * disp.cpu().double().abs()).sum(1)
        R.check("mean", mean, (exact, (130 + k) * R.U32 * size))
    leaf = obs.clone().requires_grad_()
    params = [leaf] + [q for q in net.parameters()]
    _, _, mean = predict_mixture(net, leaf, 4, mods)
    got = torch.autograd.grad(mean.square().sum(), params)
    ref = _ToyNet().to(gpu_device).double()
    leaf64 = obs.double().requires_grad_()
    top = ref.classifier(leaf64).topk(4, dim=1)
    w = top.values / top.values.sum(1, keepdim=True)
    many = leaf64.repeat_interleave(4, dim=0)
    out = ref.decoder([many, ref.synthesizer(many, labels=top.indices.reshape(-1), all_modalities=mods.double())]).reshape(29, 4, 12, 2)
    want = torch.autograd.grad((w[:, :, None, None] * out).sum(1).square().sum(), [leaf64] + [q for q in ref.parameters()])
    for a, c in zip(got, want):  # float32 sums of at most 29 * 4 * 24 terms
        assert float((a.double() - c).norm()) <= 29 * 4 * 24 * R.U32 * float(c.norm()) + 1e-12


def test_more_than_32_bits_of_scores(gpu_device):
    """2.2 M rows of 1000 scores: the last rows' elements lie beyond 2^31."""
    g = torch.Generator(device=gpu_device).manual_seed(1)
    s = torch.empty(2_200_000, 1000, dtype=torch.bfloat16, device=gpu_device).normal_(generator=g).requires_grad_()
    gw = torch.randn(2_200_000, 3, generator=g, device=gpu_device)
    ids, w = route_topk(s, 3, normalize=False)
    ds, = torch.autograd.grad(w, s, gw)
    want = R.route(s[-300:].detach().cpu(), 3, False, gw[-300:].cpu())
    assert torch.equal(ids[-300:].cpu(), want["ids"])
    R.check("w", w[-300:], want["w"])
    R.check("ds", ds[-300:], want["ds"])


def test_more_than_32_bits_of_rows(gpu_device):
    """4.4 M pairs of 512 elements there and back: places beyond 2^31 elements."""
    n, k, d = 220_000, 20, 512
    g = torch.Generator(device=gpu_device).manual_seed(2)
    plan = sort_pairs(torch.randint(0, 150, (n, k), generator=g, device=gpu_device, dtype=torch.int32), 150)
    x = torch.empty(n, d, dtype=torch.bfloat16, device=gpu_device).normal_(generator=g)
    rows = dispatch(x, plan)
    last = plan.order[-200:].long() // k
    assert torch.equal(rows[-200:], x[last])
    w = torch.rand(n, k, generator=g, device=gpu_device).requires_grad_()
    leaf = rows.requires_grad_()
    y = combine(leaf, plan, w)
    t = torch.unique(last)[:50].cpu()
    terms = rows.detach()[plan.position[t.to(gpu_device)].long()].cpu().double() * w.detach()[t.to(gpu_device)].cpu().double()[:, :, None]
    v, e32 = terms.sum(1), (k + 2) * R.U32 * terms.abs().sum(1)
    R.check("y", y[t.to(gpu_device)], (v, e32 + R.half_step(torch.bfloat16) * (v.abs() + e32)))
    gy = torch.empty(n, d, dtype=torch.bfloat16, device=gpu_device).normal_(generator=g)
    dr, dw = torch.autograd.grad(y, [leaf, w], gy)
    wl = w.detach().reshape(-1)[plan.order[-200:].long()].cpu().double()
    back = wl[:, None] * gy[last].cpu().double()
    R.check("drows", dr[-200:], (back, (R.half_step(torch.bfloat16) + 2 * R.U32) * back.abs()))
    prod = rows.detach()[-200:].cpu().double() * gy[last].cpu().double()
    R.check("dw", dw.reshape(-1)[plan.order[-200:].long()], (prod.sum(1), (d + 2) * R.U32 * prod.abs().sum(1)))


def test_capture_refuses_inputs_of_an_eager_graph(gpu_device):
    s = _scores(1, 40, 20, torch.float32).to(gpu_device).requires_grad_()
    x = torch.randn(40, 8, device=gpu_device, requires_grad=True)
    rows = torch.randn(120, 8, device=gpu_device, requires_grad=True)
    ids, w = route_topk(s, 3)  # alive, as are the next two: the leaves' nodes belong to the current stream
    plan = sort_pairs(ids, 20)
    alive = dispatch(x, plan), combine(rows, plan)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep = s.detach() * 2
        for call in (lambda: route_topk(s, 3), lambda: dispatch(x, plan), lambda: combine(rows, plan), lambda: combine(rows.detach(), plan, w)):
            with pytest.raises(RuntimeError, match="begun outside this capture"):
                call()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(keep, s.detach() * 2) and len(alive) == 2


def test_arguments_of_another_kind_are_never_taken_without_gradient(gpu_device):
    s = torch.randn(4, 8, device=gpu_device, requires_grad=True)
    plan = sort_pairs(torch.zeros(4, 1, dtype=torch.int32, device=gpu_device), 2)
    for call in (lambda: route_topk(s, 2.0), lambda: route_topk(s, "2"), lambda: combine(s, plan, [1.0]), lambda: dispatch([s], plan)):
        with pytest.raises((TypeError, ValueError)):
            call()


def test_results_of_small_calls_are_tensors_of_their_own(gpu_device):
    """They share an allocation; writing one, saving it, inference mode and gradients are as with any other tensor."""
    s = _scores(5, 12, 40, torch.float32).to(gpu_device)
    ids, w = route_topk(s, 4)
    plan = sort_pairs(ids, 40)
    kept = [t.clone() for t in (ids, w) + tuple(plan)]
    for t in (ids, w) + tuple(plan):
        assert t.is_contiguous() and t.data_ptr() % 16 == 0 and not t._is_view() and t._version == 0
        t.fill_(7)
    again = route_topk(s, 4)
    for t, k in zip(again + tuple(sort_pairs(again[0], 40)), kept):
        assert torch.equal(t, k)
    for k, t in enumerate((ids, w) + tuple(plan)):
        assert (t == 7).all(), k
    w2 = again[1].requires_grad_()
    (w2 * 2).sum().backward()
    assert (w2.grad == 2).all()
    again[0].add_(1)  # another tensor's version does not move
    assert again[1]._version == 0
    buffer = io.BytesIO()
    torch.save(again[0], buffer)
    buffer.seek(0)
    assert torch.equal(torch.load(buffer, weights_only=True), again[0])
    with torch.inference_mode():
        ids, w = route_topk(s, 4)
        assert ids.is_inference() and w.is_inference() and torch.equal(ids, kept[0]) and torch.equal(w, kept[1])
        assert torch.equal(sort_pairs(ids, 40).order, kept[3])
    rows = dispatch(torch.ones(12, 3, device=gpu_device), sort_pairs(kept[0], 40)).requires_grad_()
    combine(rows, sort_pairs(kept[0], 40), kept[1]).sum().backward()
    assert rows.grad is not None
