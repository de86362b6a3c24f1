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


def _calls(dev):
    """name -> a call of each operator that has a node, its inputs' gradients to be asked for, and the gradient of its result."""
    from pccs_accel.routing import combine, dispatch, route_topk, sort_pairs
    g = torch.Generator().manual_seed(1)

    def leaf(*shape, dtype=torch.float16):
        return torch.randn(*shape, generator=g).to(dtype).to(dev).requires_grad_()
    x, w, b, w3, b3 = leaf(40, 24), leaf(16, 24), leaf(16), leaf(5, 16, 24), leaf(5, 16)
    odd_x, odd_w = leaf(700, 97), leaf(41, 97)
    scores, rows, weights = leaf(40, 30), leaf(120, 24), leaf(40, 3, dtype=torch.float32)
    plan = sort_pairs(torch.randint(0, 30, (40, 3), generator=g, dtype=torch.int32).to(dev), 30)
    offsets = torch.tensor([0, 9, 9, 20, 30, 38], dtype=torch.int32, device=dev)
    return {
        "linear": (lambda: linear(x, w, b, "gelu"), [x, w, b]),
        "linear relu": (lambda: linear(x, w, b, "relu"), [x, w]),
        "linear odd": (lambda: linear(odd_x, odd_w, None, "silu"), [odd_x, odd_w]),
        "modality_linear": (lambda: modality_linear(x, offsets, w3, b3, "silu"), [x, w3, b3]),
        "route_topk": (lambda: route_topk(scores, 4)[1], [scores]),
        "dispatch": (lambda: dispatch(x, plan), [x]),
        "combine": (lambda: combine(rows, plan, weights), [rows, weights]),
        "combine unweighted": (lambda: combine(rows, plan), [rows]),
    }


def _backwards(t):
    """t's values in the order of a matrix stored by columns (of a vector: every other element of a longer one)."""
    return t.t().contiguous().t() if t.dim() == 2 else torch.stack((t, t), -1)[..., 0]


# what a hook may make of a tensor: another type, fewer elements, other dimensions, the host's copy, nothing, strides of its own
CHANGES = {"wider": lambda t: t.double(), "narrower": lambda t: t.to(torch.int8), "fewer rows": lambda t: t[:-1].contiguous(),
           "fewer columns": lambda t: t[..., :-1].contiguous(), "flat": lambda t: t.reshape(1, 1, 1, -1), "on the host": lambda t: t.cpu(),
           "another 16-bit type": lambda t: t.to(torch.bfloat16), "empty": lambda t: t[:0], "by columns": _backwards}


@pytest.mark.parametrize("change", list(CHANGES))
def test_saved_tensors_that_come_back_changed_are_refused(gpu_device, change):
    for name, (call, leaves) in _calls(gpu_device).items():
        kept = []
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(0) or t, lambda t: t):
            y = call()
            g = torch.ones_like(y)
            want = torch.autograd.grad(y, leaves, g)
        assert kept, name
        for which in range(len(kept)):  # each of the saved tensors in turn
            seen = []

            def unpack(t):
                seen.append(0)
                return CHANGES[change](t) if len(seen) - 1 == which else t
            with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
                y = call()
            with pytest.raises(RuntimeError, match="come back from its hook|can require gradients"):  # the latter is torch's own
                torch.autograd.grad(y, leaves, g)
        for a, c in zip(torch.autograd.grad(call(), leaves, g), want):
            assert torch.equal(a, c)


def test_views_of_negatives_are_refused_and_such_gradients_taken(gpu_device):
    """A tensor with the negative bit holds the negatives of its values; torch gives such gradients to whoever asks."""
    from pccs_accel.routing import PairPlan, combine, dispatch, route_topk, sort_pairs
    g = torch.Generator().manual_seed(2)
    x, w, b, r = (torch.randn(*s, generator=g).to(gpu_device) for s in ((40, 24), (16, 24), (16,), (40, 16)))
    ids = torch.randint(0, 9, (40, 3), generator=g, dtype=torch.int32).to(gpu_device)
    plan, weights = sort_pairs(ids, 9), torch.rand(40, 3, generator=g).to(gpu_device)
    rows = dispatch(x, plan)
    n = torch._neg_view
    for call in (lambda: linear(n(x), w), lambda: linear(x, n(w)), lambda: linear(x, w, n(b)), lambda: linear(x, w, b, None, n(r)),
                 lambda: linear(n(x[0]), w), lambda: route_topk(n(x), 3), lambda: sort_pairs(n(ids), 9), lambda: dispatch(n(x), plan),
                 lambda: combine(n(rows), plan, weights), lambda: combine(rows, plan, n(weights)),
                 lambda: dispatch(x, PairPlan(plan.offsets, plan.order, n(plan.position)))):
        with pytest.raises(ValueError, match="negative"):
            call()
    for name, (call, leaves) in _calls(gpu_device).items():
        y = call()
        gy = torch.randn(y.shape, generator=g).to(gpu_device).to(y.dtype)
        want = torch.autograd.grad(call(), leaves, -gy)
        for a, c in zip(torch.autograd.grad(y, leaves, n(gy)), want):
            assert torch.equal(a, c), name


def _has_its_own_storage(tensors):
    for t in tensors:
        assert t.storage_offset() == 0 and t.untyped_storage().nbytes() == t.numel() * t.element_size()
    assert len({t.untyped_storage().data_ptr() for t in tensors}) == len(tensors)


def test_results_and_gradients_grow_and_go_by_themselves(gpu_device):
    """resize_ (and out= with another shape) of one result leaves the others as they are."""
    from pccs_accel.routing import combine, dispatch, route_topk, sort_pairs
    g = torch.Generator().manual_seed(4)
    scores = torch.randn(12, 40, generator=g).to(gpu_device).requires_grad_()
    x = torch.randn(12, 8, generator=g).to(gpu_device).requires_grad_()
    w = torch.randn(6, 8, generator=g).to(gpu_device).requires_grad_()
    b = torch.randn(6, generator=g).to(gpu_device).requires_grad_()
    ids, weights = route_topk(scores, 4)
    plan = sort_pairs(ids, 40)
    rows = dispatch(x, plan)
    y = linear(x, w, b, "gelu")
    rows2 = rows.detach().requires_grad_()
    mean = combine(rows2, plan, weights)
    results = [ids, weights, *plan, rows, y, mean]
    grads = list(torch.autograd.grad([y, mean], [x, w, b, rows2, scores], [torch.ones_like(y), torch.ones_like(mean)]))
    every = [t.detach() for t in results + grads]
    _has_its_own_storage(every)
    kept = [t.clone() for t in every]
    for i, t in enumerate(every):
        t.resize_(t.numel() + 4096).fill_(-7)
        for other, value in list(zip(every, kept))[i + 1:]:
            assert torch.equal(other, value)
        t.untyped_storage().resize_(0)
