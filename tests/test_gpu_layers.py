"""``pccs_accel.layers`` on the GPU against float64 formulas (routing_reference.py: element-wise bounds that count roundings)."""
import itertools

import pytest
import torch
import torch.utils.checkpoint

import routing_reference as R
from pccs_accel import kernels as K
from pccs_accel.layers import linear, modality_linear

pytestmark = pytest.mark.gpu


def _inputs(seed, rows, i, o, dtype, lead=(), bias=True, residual=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.tanh(torch.randn(rows, i, generator=g)).to(dtype)
    w = (torch.randn(lead + (o, i), generator=g) / i ** 0.5).to(dtype)
    b = (torch.randn(lead + (o,), generator=g) * 0.1).to(dtype) if bias else None
    r = torch.randn(rows, o, generator=g).to(dtype) if residual else None
    gy = torch.randn(rows, o, generator=g).to(dtype)
    return x, w, b, r, gy


def _run(dev, x, w, b, r, gy, act, offsets=None):
    leaves = [t.to(dev).requires_grad_() if t is not None else None for t in (x, w, b, r)]
    if offsets is None:
        y = linear(leaves[0], leaves[1], leaves[2], activation=act, residual=leaves[3])
    else:
        y = modality_linear(leaves[0], offsets.to(dev), leaves[1], leaves[2], activation=act, residual=leaves[3])
    have = [t for t in leaves if t is not None]
    grads = iter(torch.autograd.grad(y, have, gy.to(dev)))
    got = {"y": y}
    for name, t in zip(("dx", "dw", "db", "dres"), leaves):
        if t is not None:
            got[name] = next(grads)
    return got


def _compare(got, want, dtype):
    for name, v in got.items():
        assert v.dtype == dtype, name
        R.check(name, v, want[name])


# rows, in, out: one token, tiles' edges, sizes nothing divides, a long sum, more rows than one wave of tiles
SIZES = [(1, 1, 1), (1, 96, 200), (3, 7, 5), (16, 48, 24), (17, 97, 201), (33, 130, 31), (64, 64, 64), (65, 63, 129),
         (127, 256, 96), (300, 33, 257), (512, 1025, 40), (2614, 96, 200)]


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_linear_and_gradients(gpu_device, size, dtype):
    acts = [None, "relu", "gelu", "silu"]
    n = SIZES.index(size)
    x, w, b, r, gy = _inputs(n, *size, dtype, bias=n % 3 != 1, residual=n % 2 == 0)
    act = acts[(n + R.TYPES.index(dtype)) % 4]
    _compare(_run(gpu_device, x, w, b, r, gy, act), R.linear(x, w, b, act, r, gy), dtype)


@pytest.mark.parametrize("act,bias,residual", list(itertools.product([None, "relu", "gelu", "silu"], [False, True], [False, True])))
def test_linear_epilogues(gpu_device, act, bias, residual):
    for dtype in R.TYPES:
        x, w, b, r, gy = _inputs(5, 70, 72, 66, dtype, bias=bias, residual=residual)
        _compare(_run(gpu_device, x, w, b, r, gy, act), R.linear(x, w, b, act, r, gy), dtype)


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
@pytest.mark.parametrize("size", [(40000, 24, 40), (20000, 130, 300), (33000, 8, 8)], ids=str)
def test_linear_many_rows(gpu_device, size, dtype):
    """Big tiles forward, and a weight gradient summed in parts."""
    x, w, b, r, gy = _inputs(9, *size, dtype, residual=False)
    _compare(_run(gpu_device, x, w, b, r, gy, "gelu"), R.linear(x, w, b, "gelu", r, gy), dtype)


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
@pytest.mark.parametrize("rows", [1, 2, 15, 16, 17, 32, 33, 64, 65])
def test_linear_few_rows(gpu_device, rows, dtype):
    """The kernels for few rows and their borders: long sums, sizes and row starts of every alignment."""
    for i, o, start in ((1024, 1024, 0), (511, 33, 0), (130, 7, 1), (31, 16, 3), (2048, 40, 5)):
        x, w, b, r, _ = _inputs(rows + i, rows, i + 8, o, dtype)
        x, w = x[:, start:start + i], w[:, :i].contiguous()
        y = linear(_strided(x, gpu_device), w.to(gpu_device), b.to(gpu_device), "gelu", r.to(gpu_device))
        R.check("y", y, R.linear(x, w, b, "gelu", r)["y"])


def _strided(x, dev):
    """x on the device with the strides it has."""
    whole = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device=dev)
    return whole.copy_(x)


def test_linear_wide(gpu_device):
    for dtype in R.TYPES:
        x, w, b, r, gy = _inputs(11, 700, 1200, 1100, dtype)
        _compare(_run(gpu_device, x, w, b, r, gy, "silu"), R.linear(x, w, b, "silu", r, gy), dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
def test_which_rows_are_laid_out_anew(gpu_device, dtype):
    """x, the weights, the gradient or none of them start where the products want them; one row of output; with and without sets."""
    for i, o, slice_x, act in ((64, 41, True, None), (97, 40, False, None), (97, 41, True, "silu"), (33, 1, False, None), (32, 1, True, "relu")):
        x, w, b, r, gy = _inputs(i + o, 300, i, o, dtype, residual=False)
        if slice_x:
            x = torch.cat([x[:, :1], x], 1)[:, 1:]  # rows i + 1 apart, from the second element on
        leaves = [_strided(x, gpu_device) if slice_x else x.to(gpu_device), w.to(gpu_device), b.to(gpu_device)]
        if o == 1:  # contiguous, whatever distance its only row names
            leaves[1] = torch.cat([leaves[1], leaves[1]], 1)[:, :i]
            assert leaves[1].is_contiguous() and leaves[1].stride(0) == 2 * i
        got = [t.requires_grad_() for t in leaves]
        y = linear(*got, activation=act)
        grads = torch.autograd.grad(y, got, gy.to(gpu_device))
        _compare(dict(zip(("y", "dx", "dw", "db"), (y,) + grads)), R.linear(x, w, b, act, None, gy), dtype)
        offsets = torch.tensor([0, 100, 100, 290], dtype=torch.int32)
        x, w, b, r, gy = _inputs(i + o + 1, 300, i, o, dtype, residual=False, lead=(3,))
        _compare(_run(gpu_device, x, w, b, None, gy, act, offsets), R.modality_linear(x, offsets, w, b, act, None, gy), dtype)


@pytest.mark.parametrize("dtype,act", [(torch.bfloat16, "gelu"), (torch.float16, "silu")], ids=str)
def test_linear_that_fills_the_card(gpu_device, dtype, act):
    """The largest tiles in all three products, ragged on every side."""
    x, w, b, r, gy = _inputs(15, 8200, 1801, 1797, dtype)
    _compare(_run(gpu_device, x, w, b, r, gy, act), R.linear(x, w, b, act, r, gy), dtype)


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
def test_linear_takes_slices_and_odd_addresses(gpu_device, dtype):
    """The observation half of a memory [N, obs + pred] is a slice of columns; an odd column start is no multiple of 4 bytes."""
    dev = gpu_device
    g = torch.Generator().manual_seed(3)
    memory = torch.randn(90, 131, generator=g).to(dtype)
    w = torch.randn(50, 48, generator=g).to(dtype)
    wide = torch.randn(90, 77, generator=g).to(dtype)
    for start in (0, 1, 2, 48, 83):
        x, r = memory[:, start:start + 48], wide[:, start % 27:start % 27 + 50]
        y = linear(memory.to(dev)[:, start:start + 48], w.to(dev), residual=wide.to(dev)[:, start % 27:start % 27 + 50])
        R.check("y", y, R.linear(x, w, None, None, r)["y"])
    flat = torch.randn(50 * 48 + 1, generator=g).to(dtype)
    y = linear(memory.to(dev)[:, :48], flat.to(dev)[1:].view(50, 48))
    R.check("y", y, R.linear(memory[:, :48], flat[1:].view(50, 48), None, None, None)["y"])


def test_linear_of_more_dimensions(gpu_device):
    x, w, b, r, _ = _inputs(4, 30, 40, 50, torch.float32)
    want = R.linear(x, w, b, "gelu", r)["y"]
    y = linear(x.to(gpu_device).view(5, 6, 40), w.to(gpu_device), b.to(gpu_device), "gelu", r.to(gpu_device).view(5, 6, 50))
    assert y.shape == (5, 6, 50)
    R.check("y", y.view(30, 50), want)
    y = linear(x.to(gpu_device)[0], w.to(gpu_device), b.to(gpu_device), "gelu", r.to(gpu_device)[0])
    assert y.shape == (50,)
    assert linear(x.to(gpu_device)[:0], w.to(gpu_device)).shape == (0, 50)
    assert linear(x.to(gpu_device).view(5, 6, 40)[:0], w.to(gpu_device)).shape == (0, 6, 50)


def test_linear_gradients_against_differences(gpu_device):
    """Float32, central differences of sum(g * y) along random directions in float64 inputs rounded to float32."""
    for act in ("gelu", "silu"):
        x, w, b, r, gy = _inputs(21, 40, 30, 20, torch.float32)
        got = _run(gpu_device, x, w, b, r, gy, act)
        gen = torch.Generator().manual_seed(1)
        for name, t in (("dx", x), ("dw", w), ("db", b)):
            d = torch.randn(t.shape, generator=gen, dtype=torch.float64)
            h = 1e-4

            def value(step):
                p = {"dx": x.double(), "dw": w.double(), "db": b.double()}
                p[name] = p[name] + step * d
                return float((gy.double() * (R.act(p["dx"] @ p["dw"].T + p["db"], act))).sum())
            slope = (value(h) - value(-h)) / (2 * h)
            mine = got[name].detach().cpu().double()
            # h^2 / 6 of the third derivative, and the float32 gradient's own error (element bounds, added up)
            err = float((R.linear(x, w, b, act, r, gy)[name][1] * d.abs()).sum()) + 1e-5 * float((mine * d).abs().sum())
            assert abs(slope - float((mine * d).sum())) <= err, (act, name)


def test_linear_keeps_nan_and_infinity(gpu_device):
    for dtype in R.TYPES:
        for act in (None, "relu", "gelu", "silu"):
            x = torch.ones(70, 9, dtype=dtype)
            x[3, 2] = float("nan")
            x[5, 1] = float("inf")
            w = torch.ones(6, 9, dtype=dtype)
            y = linear(x.to(gpu_device), w.to(gpu_device), activation=act).cpu().float()
            assert torch.isnan(y[3]).all() and torch.isinf(y[5]).all()
            keep = torch.ones(70, dtype=torch.bool)
            keep[[3, 5]] = False
            assert torch.isfinite(y[keep]).all()


def test_linear_neighbours_do_not_leak(gpu_device):
    """What lies beside the rows and behind the sums is NaN: nothing of it may reach a result."""
    for dtype in R.TYPES:
        for i, o, n in ((50, 30, 37), (96, 64, 64), (33, 17, 200)):
            big = torch.full((n + 4, i + 40), float("nan"), dtype=dtype)
            g = torch.Generator().manual_seed(i)
            x = torch.randn(n, i, generator=g).to(dtype)
            big[2:n + 2, 8:i + 8] = x
            w = torch.randn(o, i, generator=g).to(dtype)
            r = torch.randn(n, o, generator=g).to(dtype)
            gy = torch.randn(n, o, generator=g).to(dtype)
            xd = big.to(gpu_device)[2:n + 2, 8:i + 8].requires_grad_()
            wd = w.to(gpu_device).requires_grad_()
            y = linear(xd, wd, activation="relu", residual=r.to(gpu_device))
            dx, dw = torch.autograd.grad(y, [xd, wd], gy.to(gpu_device))
            want = R.linear(x, w, None, "relu", r, gy)
            for name, v in (("y", y), ("dx", dx), ("dw", dw)):
                R.check(name, v, want[name])


def _offsets(seed, rows, sets, behind=0, empty=0.3):
    g = torch.Generator().manual_seed(seed)
    share = torch.rand(sets, generator=g) * (torch.rand(sets, generator=g) > empty)
    if float(share.sum()) == 0:
        share[sets // 2] = 1
    who = torch.multinomial(share, rows - behind, replacement=True, generator=g) if rows > behind else torch.zeros(0).long()
    return torch.cat([torch.zeros(1).long(), torch.bincount(who, minlength=sets).cumsum(0)]).to(torch.int32)


# rows, in, out, modalities, rows behind the last one
SETS = [(1, 8, 8, 1, 0), (1, 96, 24, 200, 0), (5, 7, 9, 3, 2), (64, 128, 512, 200, 0), (200, 33, 65, 7, 31), (130, 96, 64, 65, 0),
        (300, 40, 24, 128, 299), (2000, 96, 130, 12, 77), (4000, 24, 36, 200, 0), (6000, 97, 33, 5, 1)]


@pytest.mark.parametrize("dtype", R.TYPES, ids=str)
@pytest.mark.parametrize("size", SETS, ids=str)
def test_modality_linear_and_gradients(gpu_device, size, dtype):
    rows, i, o, sets, behind = size
    n = SETS.index(size)
    x, w, b, r, gy = _inputs(n, rows, i, o, dtype, lead=(sets,), bias=n % 3 != 1, residual=n % 2 == 0)
    offsets = _offsets(n, rows, sets, behind)
    act = [None, "relu", "gelu", "silu"][(n + R.TYPES.index(dtype)) % 4]
    if behind:
        x[rows - behind:] = float("nan")  # never read into a result
    _compare(_run(gpu_device, x, w, b, r, gy, act, offsets), R.modality_linear(x, offsets, w, b, act, r, gy), dtype)


def test_modality_linear_all_rows_behind(gpu_device):
    x, w, b, r, gy = _inputs(1, 70, 16, 24, torch.bfloat16, lead=(4,))
    offsets = torch.zeros(5, dtype=torch.int32)
    got = _run(gpu_device, x, w, b, r, gy, "gelu", offsets)
    for name, v in got.items():
        assert not v.any(), name


def test_modality_linear_many_sets(gpu_device):
    x, w, b, r, gy = _inputs(2, 3000, 16, 8, torch.float32, lead=(1000,))
    offsets = _offsets(7, 3000, 1000)
    _compare(_run(gpu_device, x, w, b, r, gy, "silu", offsets), R.modality_linear(x, offsets, w, b, "silu", r, gy), torch.float32)


def test_modality_linear_survives_bad_offsets(gpu_device):
    """Offsets that leave the rows or decrease are the caller's mistake; nothing outside the tensors is touched."""
    x, w, b, _, _ = _inputs(3, 50, 16, 8, torch.float32, lead=(3,))
    for bad in ([0, 1000, 2000, 3000], [-5, 10, 20, 1 << 30], [0, 40, 10, 50], [50, 50, 50, 50]):
        y = modality_linear(x.to(gpu_device), torch.tensor(bad, dtype=torch.int32, device=gpu_device), w.to(gpu_device), b.to(gpu_device))
        torch.cuda.synchronize()
        assert y.shape == (50, 8)


def test_some_gradients_only(gpu_device):
    x, w, b, r, gy = _inputs(8, 90, 20, 30, torch.float32)
    want = R.linear(x, w, b, "gelu", r, gy)
    d = gpu_device
    for needs in itertools.product([False, True], repeat=4):
        if not any(needs):
            continue
        leaves = [t.to(d).requires_grad_(n) for t, n in zip((x, w, b, r), needs)]
        y = linear(leaves[0], leaves[1], leaves[2], "gelu", leaves[3])
        asked = [t for t in leaves if t.requires_grad]
        grads = iter(torch.autograd.grad(y, asked, gy.to(d)))
        for name, t in zip(("dx", "dw", "db", "dres"), leaves):
            if t.requires_grad:
                R.check(name, next(grads), want[name])


def test_same_tensor_twice_and_broadcast_gradient(gpu_device):
    """x as its own residual; a gradient that is an expanded scalar."""
    x, w, b, _, _ = _inputs(12, 40, 32, 32, torch.float32)
    xd, wd = x.to(gpu_device).requires_grad_(), w.to(gpu_device).requires_grad_()
    y = linear(xd, wd, b.to(gpu_device), "silu", xd)
    dx, dw = torch.autograd.grad(y.sum(), [xd, wd])
    want = R.linear(x, w, b, "silu", x, torch.ones(40, 32))
    R.check("y", y, want["y"])
    v, e = want["dx"]
    R.check("dx", dx, (v + 1, e + 2 * R.U32 * (v.abs() + 1)))
    R.check("dw", dw, want["dw"])


def test_results_repeat_bit_for_bit(gpu_device):
    x, w, b, r, gy = _inputs(13, 30000, 96, 72, torch.bfloat16)
    first = _run(gpu_device, x, w, b, r, gy, "gelu")
    for _ in range(3):
        again = _run(gpu_device, x, w, b, r, gy, "gelu")
        for name in first:
            assert torch.equal(first[name], again[name]), name


def test_on_another_stream_and_in_a_graph(gpu_device):
    x, w, b, r, gy = (t.to(gpu_device) for t in _inputs(14, 333, 96, 104, torch.bfloat16))
    want = linear(x, w, b, "gelu", r)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = linear(x, w, b, "gelu", r)
    side.synchronize()
    assert torch.equal(y, want)

    def step(x, w, b, r, gy):
        y, pre = K.linear(x, w, b, "gelu", r, want_pre=True)
        dz = K.linear_act_grad(gy, pre, "gelu")
        return (y, K.linear_grad_input(dz, w)) + K.linear_grad_weight(dz, x, want_bias=True)
    graphs = []
    for _ in range(2):
        static = [t.clone() for t in (x, w, b, r, gy)]
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(*static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(*static)
        graphs.append((graph, static, outs))
    for turn in range(4):
        for graph, static, outs in graphs:
            for t, src in zip(static, (x, w, b, r, gy)):
                t.copy_(src * (turn + 1) / 2)
            graph.replay()
            torch.cuda.synchronize()
            eager = step(*[t.clone() for t in static])
            for a, c in zip(outs, eager):
                assert torch.equal(a, c)


def test_backward_in_a_graph(gpu_device):
    x, w, b, r, gy = (t.to(gpu_device) for t in _inputs(15, 200, 48, 40, torch.float32))
    leaves = [t.requires_grad_() for t in (x, w, b, r)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            torch.autograd.grad(linear(leaves[0], leaves[1], leaves[2], "gelu", leaves[3]), leaves, gy)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = linear(leaves[0], leaves[1], leaves[2], "gelu", leaves[3])
        grads = torch.autograd.grad(y, leaves, gy)
    for turn in range(3):
        with torch.no_grad():
            x.mul_(0.9)
            gy.mul_(-1.1)
        graph.replay()
        torch.cuda.synchronize()
        fresh = [t.detach().clone().requires_grad_() for t in leaves]
        eager = torch.autograd.grad(linear(fresh[0], fresh[1], fresh[2], "gelu", fresh[3]), fresh, gy)
        for a, c in zip(grads, eager):
            assert torch.equal(a, c)


def test_refusals(gpu_device):
    d = gpu_device
    x, w = torch.zeros(4, 8, device=d), torch.zeros(6, 8, device=d)
    w3, off = torch.zeros(2, 6, 8, device=d), torch.tensor([0, 2, 4], dtype=torch.int32, device=d)
    for call, error in [
        (lambda: linear(x, w.double()), TypeError),
        (lambda: linear(x.double(), w.double()), TypeError),
        (lambda: linear(x, w.half()), TypeError),
        (lambda: linear(x, w[:, :7]), ValueError),
        (lambda: linear(x[:, :7], w), ValueError),
        (lambda: linear(x, w.T), ValueError),
        (lambda: linear(x.T.contiguous().T, w), ValueError),
        (lambda: linear(x[:1].expand(4, 8), w), ValueError),
        (lambda: linear(x, w, torch.zeros(5, device=d)), ValueError),
        (lambda: linear(x, w, torch.zeros(6, device=d, dtype=torch.float16)), TypeError),
        (lambda: linear(x, w, residual=torch.zeros(4, 5, device=d)), ValueError),
        (lambda: linear(x, w, activation="tanh"), ValueError),
        (lambda: linear(x, torch.zeros(6, 0, device=d)), ValueError),
        (lambda: linear(x.cpu(), w), K._lib.MtpError),
        (lambda: linear(x, w.cpu()), K._lib.MtpError),
        (lambda: linear(x, None), TypeError),
        (lambda: modality_linear(x, None, w3), TypeError),
        (lambda: modality_linear(x, off.long(), w3), TypeError),
        (lambda: modality_linear(x, off[:2], w3), ValueError),
        (lambda: modality_linear(x, off, w), ValueError),
        (lambda: modality_linear(x, off, w3, torch.zeros(6, device=d)), ValueError),
    ]:
        with pytest.raises(error):
            call()


def test_second_derivatives_are_refused(gpu_device):
    x, w, b, r, gy = (t.to(gpu_device) for t in _inputs(16, 20, 8, 8, torch.float32))
    x, w = x.requires_grad_(), w.requires_grad_()
    y = linear(x, w, b, "gelu")
    dx, = torch.autograd.grad(y, x, gy, create_graph=True)
    R.check("dx", dx, R.linear(x.detach().cpu(), w.detach().cpu(), b.cpu(), "gelu", None, gy.cpu())["dx"])
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(dx.sum(), x)


def test_rows_laid_out_anew_keep_the_inputs_history(gpu_device):
    """Odd 16-bit rows: both passes use a copy of x and of the weights, and the node still knows where they came from."""
    x, w, b, r, gy = (t.to(gpu_device) for t in _inputs(18, 600, 97, 41, torch.float16))
    x, w = x.requires_grad_(), w.requires_grad_()
    y = linear(x, w, b, "gelu")
    dx, = torch.autograd.grad(y, x, gy, create_graph=True)
    R.check("dx", dx, R.linear(x.detach().cpu(), w.detach().cpu(), b.cpu(), "gelu", None, gy.cpu())["dx"])
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(dx.float().sum(), w)
    for t in (x, w):
        y = linear(x, w, b, "gelu")
        with torch.no_grad():
            t.mul_(2)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, x, gy)


def test_changed_inputs_are_noticed_by_the_backward_pass(gpu_device):
    x, w, b, r, gy = (t.to(gpu_device) for t in _inputs(17, 20, 8, 8, torch.float32))
    x = x.requires_grad_()
    y = linear(x, w, b, "relu")
    y.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, gy)
    y = linear(x, w, b, "gelu")
    w.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, gy)


def test_front_ends_and_nodes_agree_bit_for_bit(gpu_device):
    """The entry points through ``kernels`` (no autograd) and through the nodes."""
    for dtype in R.TYPES:
        x, w, b, r, gy = (t.to(gpu_device) for t in _inputs(18, 1500, 40, 56, dtype))
        leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
        y = linear(leaves[0], leaves[1], leaves[2], "silu", leaves[3])
        dx, dw, db, dr = torch.autograd.grad(y, leaves, gy)
        y2, pre = K.linear(x, w, b, "silu", r, want_pre=True)
        dx2, dw2, db2 = K.linear_backward(gy, pre, "silu", x, w)
        for a, c in ((y, y2), (dx, dx2), (dw, dw2), (db, db2), (dr, gy)):
            assert torch.equal(a, c)


def test_no_rows_still_have_gradients(gpu_device):
    for dtype in R.TYPES:
        x, w, b, r, gy = _inputs(19, 0, 9, 7, dtype)
        got = _run(gpu_device, x, w, b, r, gy, "gelu")
        assert got["y"].shape == (0, 7) and got["dx"].shape == (0, 9)
        assert not got["dw"].any() and not got["db"].any() and got["dw"].shape == (7, 9)
        x, w, b, r, gy = _inputs(19, 0, 9, 7, dtype, lead=(3,))
        got = _run(gpu_device, x, w, b, r, gy, "relu", torch.zeros(4, dtype=torch.int32))
        assert not got["dw"].any() and not got["db"].any() and got["dw"].shape == (3, 7, 9)


def test_more_than_32_bits_of_elements(gpu_device):
    """1.1 M rows of 2048: the last rows' elements lie beyond 2^31, their bytes beyond 2^32."""
    n, i, o, tail = 1_100_000, 2048, 8, 40
    g = torch.Generator(device=gpu_device).manual_seed(1)
    x = torch.empty(n, i, dtype=torch.bfloat16, device=gpu_device).normal_(generator=g).requires_grad_()
    w = (torch.randn(o, i, generator=g, device=gpu_device) / 45).to(torch.bfloat16).requires_grad_()
    gy = torch.zeros(n, o, dtype=torch.bfloat16, device=gpu_device)
    gy[-tail:] = torch.randn(tail, o, generator=g, device=gpu_device).to(torch.bfloat16)
    y = linear(x, w, activation="gelu")
    dx, dw = torch.autograd.grad(y, [x, w], gy)
    want = R.linear(x[-tail:].detach().cpu(), w.detach().cpu(), None, "gelu", None, gy[-tail:].cpu())
    R.check("y", y[-tail:], want["y"])
    R.check("dx", dx[-tail:], want["dx"])
    R.check("dw", dw, want["dw"])
    assert not dx[:-tail].any()
    # the same the other way round: a wide output
    x2, w2 = gy[:, :8].contiguous(), x[:2048, :8].detach().contiguous()
    y2 = linear(x2, w2)
    R.check("y2", y2[-tail:], R.linear(x2[-tail:].cpu(), w2.cpu(), None, None, None)["y"])
    assert not y2[:-tail].any()


def test_capture_refuses_inputs_of_an_eager_graph(gpu_device):
    x, w, b, r, gy = (t.to(gpu_device) for t in _inputs(20, 40, 16, 8, torch.float32))
    w = w.requires_grad_()
    eager = linear(x, w, b, "gelu")  # alive: w's node belongs to the current stream
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        keep = x * 2  # something to capture
        with pytest.raises(RuntimeError, match="begun outside this capture"):
            linear(x, w, b, "gelu")
        with torch.no_grad():
            inner = linear(x, w, b, "gelu")  # no backward pass: fine
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(inner, eager) and torch.equal(keep, x * 2)


def test_arguments_of_another_kind_are_never_taken_without_gradient(gpu_device):
    x = torch.randn(4, 8, device=gpu_device, requires_grad=True)
    for call in (lambda: linear(x, [1.0]), lambda: linear(x, 3), lambda: linear(x, x, bias="b")):
        with pytest.raises((TypeError, ValueError)):
            call()


def test_no_rows_and_only_the_inputs_gradient(gpu_device):
    x = torch.zeros(0, 8, device=gpu_device, requires_grad=True)
    w = torch.randn(5, 8, device=gpu_device)
    dx, = torch.autograd.grad(linear(x, w, activation="gelu"), x, torch.zeros(0, 5, device=gpu_device))
    assert dx.shape == (0, 8)


def test_nodes_behave_like_torchs(gpu_device):
    """Twice through a graph, kept or not; hooks; a leaf's .grad; undefined gradients; forward mode is refused, not forgotten."""
    x, w, b, r, gy = (t.to(gpu_device) for t in _inputs(30, 50, 12, 9, torch.float32))
    for act in (None, "relu", "silu"):
        leaves = [t.clone().requires_grad_() for t in (x, w, b, r)]
        y = linear(leaves[0], leaves[1], leaves[2], act, leaves[3])
        assert y.grad_fn is not None and "Linear" in y.grad_fn.name()
        once = torch.autograd.grad(y, leaves, gy, retain_graph=True)
        again = torch.autograd.grad(y, leaves, gy)
        assert all(torch.equal(p, q) for p, q in zip(once, again))
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y, leaves, gy)
        seen = []
        leaves[1].register_hook(lambda g: seen.append(g.clone()))
        (linear(leaves[0], leaves[1], leaves[2], act, leaves[3]) * gy).sum().backward()
        assert len(seen) == 1 and torch.equal(seen[0], leaves[1].grad)
        assert all(torch.equal(t.grad, g) for t, g in zip(leaves, once))
        (linear(leaves[0], leaves[1], leaves[2], act, leaves[3]) * gy).sum().backward()  # added to what is there
        assert all(torch.equal(t.grad, 2 * g) for t, g in zip(leaves, once))
    y = linear(leaves[0], leaves[1].detach())
    z = linear(y, torch.ones(4, 9, device=gpu_device))
    assert leaves[0].grad.add_(1)._version  # small gradients share an allocation: the others are left as they are
    assert torch.equal(leaves[1].grad, 2 * once[1]) and torch.equal(leaves[2].grad, 2 * once[2])
    del y
    z.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="forward mode"):
            linear(dual, w)


@pytest.mark.parametrize("sizes", [(300, 97, 41), (300, 96, 40), (20, 33, 7)], ids=str)
def test_hooks_on_saved_tensors(gpu_device, sizes):
    """Saved tensors that go to the host and come back have other strides than those that went; recomputed ones are new."""
    for dtype, act in ((torch.float16, "gelu"), (torch.bfloat16, "relu"), (torch.float32, "silu")):
        x, w, b, r, gy = _inputs(sum(sizes), *sizes, dtype, residual=False)
        wide = torch.cat([x, x], 1).to(gpu_device)
        leaves = [wide[:, :sizes[1]].requires_grad_(), w.to(gpu_device).requires_grad_(), b.to(gpu_device).requires_grad_()]
        want = torch.autograd.grad(linear(*leaves, activation=act), leaves, gy.to(gpu_device))
        with torch.autograd.graph.save_on_cpu():
            y = linear(*leaves, activation=act)
        for got, expected in zip(torch.autograd.grad(y, leaves, gy.to(gpu_device)), want):
            assert torch.equal(got, expected)
        y = torch.utils.checkpoint.checkpoint(lambda *a: linear(*a, activation=act), *leaves, use_reentrant=False)
        for got, expected in zip(torch.autograd.grad(y, leaves, gy.to(gpu_device)), want):
            assert torch.equal(got, expected)


def test_hooks_that_change_a_layout_are_refused(gpu_device):
    x, w, b, r, gy = (t.to(gpu_device) for t in _inputs(31, 40, 16, 12, torch.float32))
    w.requires_grad_()
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.t().contiguous().t() if t.dim() == 2 else t):
        y = linear(x, w, b, "gelu")
    with pytest.raises(RuntimeError, match="another layout"):
        torch.autograd.grad(y, w, gy)
