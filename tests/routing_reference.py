"""The router, the pair sort and the linear layers in float64 on the CPU, with error bounds for the kernels' results.

Bounds count roundings: u is half a step of a type relative to the value (float32 2^-24, bfloat16 2^-8 / 2, ...: eps / 2), a sum
of m float32 terms is off by at most about m u32 times the sum of the terms' magnitudes, whatever its order."""
import math

import torch

U32 = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def floor_of(dtype):
    """Half the distance of the type's smallest numbers: what a rounding near zero can cost."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def act(z, kind):
    if kind == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if kind == "gelu":
        return 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
    if kind == "silu":
        return z * torch.sigmoid(z)
    return z


def slope(z, kind):
    if kind == "relu":
        return (z > 0).double()
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(z / math.sqrt(2))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if kind == "silu":
        q = torch.sigmoid(z)
        return q * (1 + z * (1 - q))
    return torch.ones_like(z)


# largest second derivative of the activation: gelu 2 / sqrt(2 pi) at 0, silu 1/2 at 0
BEND = {"gelu": 0.8, "silu": 0.5, "relu": 0.0, None: 0.0}


def linear(x, w, b, kind, res, g=None):
    """dict(name -> (value, bound)) of y, dx, dw, db, dres for one weight matrix; inputs in the kernels' type, on the CPU."""
    t = x.dtype
    u = half_step(t)
    X, W = x.double(), w.double()
    B = b.double() if b is not None else torch.zeros(w.shape[0], dtype=torch.float64)
    k = X.shape[1]
    z = X @ W.T + B
    size = X.abs() @ W.abs().T + B.abs()
    ez = (k + 2) * U32 * size
    y = act(z, kind)
    R = res.double() if res is not None else torch.zeros_like(y)
    # activations change by at most 1.13 times the change of z; erf, exp and the products around them: 8 roundings of z
    ey = 1.13 * ez + 8 * U32 * z.abs() + 2 * U32 * (y.abs() + R.abs())
    out = {"y": (y + R, ey + u * ((y + R).abs() + ey) + floor_of(t))}
    if g is None:
        return out
    G = g.double()
    s = slope(z, kind)
    # z is kept in the type: its rounding (and that of its computation) moves the slope by at most BEND times as much
    moved = ez + u * (z.abs() + ez) + floor_of(t)
    ez_slope = BEND[kind] * moved + (8 * U32 * (1 + z.abs()) if kind in ("gelu", "silu") else 0.0)
    if kind == "relu":  # where z may have another sign the slope may be the other one
        ez_slope = (z.abs() <= ez).double()
    dz = G * s
    edz = G.abs() * ez_slope
    if kind is not None:
        edz = edz + (u + 2 * U32) * (dz.abs() + edz) + floor_of(t)
    n, o = X.shape[0], W.shape[0]
    dx, ex = dz @ W, edz @ W.abs() + (o + 2) * U32 * ((dz.abs() + edz) @ W.abs())
    dw, ew = dz.T @ X, edz.T @ X.abs() + (n + 2) * U32 * ((dz.abs() + edz).T @ X.abs())
    db, eb = dz.sum(0), edz.sum(0) + (n + 2) * U32 * (dz.abs() + edz).sum(0)
    for name, v, e in (("dx", dx, ex), ("dw", dw, ew), ("db", db, eb)):
        out[name] = (v, e + u * (v.abs() + e) + floor_of(t))
    out["dres"] = (G, torch.zeros_like(G))
    return out


def modality_linear(x, offsets, w, b, kind, res, g=None):
    """The same with one matrix per modality; rows behind offsets[-1] are zeros without gradient."""
    at = offsets.tolist()
    n, (s, o, i) = x.shape[0], w.shape
    shapes = {"y": (n, o), "dx": (n, i), "dw": (s, o, i), "db": (s, o), "dres": (n, o)}
    out = {k: (torch.zeros(v, dtype=torch.float64), torch.zeros(v, dtype=torch.float64)) for k, v in shapes.items()}
    for e in range(s):
        lo, hi = at[e], at[e + 1]
        if hi == lo:
            continue
        part = linear(x[lo:hi], w[e], b[e] if b is not None else None, kind, res[lo:hi] if res is not None else None,
                      g[lo:hi] if g is not None else None)
        for name, (v, err) in part.items():
            where = e if name in ("dw", "db") else slice(lo, hi)
            out[name][0][where] = v
            out[name][1][where] = err
    return out


def route(scores, k, normalize, g=None):
    """ids, and (value, bound) of the weights and of the scores' gradient."""
    s = scores.double()
    n, e = s.shape
    clean = torch.where(torch.isnan(s), torch.full_like(s, -math.inf), s)
    order = torch.sort(clean, dim=1, descending=True, stable=True).indices[:, :k]
    picked = clean.gather(1, order)
    ids = torch.where(picked == -math.inf, torch.full_like(order, -1), order)
    top = clean.max(1, keepdim=True).values
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp(clean - top)
    mass = torch.exp(picked - top).sum(1, keepdim=True) if normalize else p.sum(1, keepdim=True)
    p = torch.where(mass > 0, p / mass, torch.zeros_like(p))
    w = torch.where(ids >= 0, p.gather(1, order), torch.zeros_like(picked))
    # exponents are differences of scores, rounded once (u32 |s - top|); exp, the sum over e (or k) terms and the division
    gap = torch.where(torch.isfinite(clean), (clean - top).abs(), torch.zeros_like(clean))
    rel = (4 * gap.max(1, keepdim=True).values.clamp_max(104.0) + (k if normalize else e) + 12) * U32
    bad = torch.isnan(s).any(1)
    w[bad] = math.nan
    out = {"ids": ids.to(torch.int32), "w": (w, rel * w.abs() + 1e-38)}
    if g is not None:
        G = g.double()
        u = half_step(scores.dtype)
        dot, size = (w * G).sum(1, keepdim=True), (w * G).abs().sum(1, keepdim=True)
        back = torch.zeros_like(s).scatter_add(1, ids.clamp_min(0).to(torch.int64), torch.where(ids >= 0, w * G, torch.zeros_like(w)))
        mine = torch.zeros_like(s).scatter_add(1, ids.clamp_min(0).to(torch.int64), torch.where(ids >= 0, w, torch.zeros_like(w)))
        weight = mine if normalize else p
        v = back - weight * dot
        err = (2 * rel + (k + 4) * U32) * (back.abs() + weight * size)
        # below the smallest normal float a rounding costs up to half of 2^-149 whatever the value: one in exp(s - top), one in the
        # weight made of it (the scale 1 / mass is at most 1, as the largest term is exp(0)), both then multiplied by g - dot or
        # dot, and one in that product
        low = floor_of(torch.float32) * (1 + 2 * (G.abs().max(1, keepdim=True).values + size))
        out["ds"] = (v, err + low + u * (v.abs() + err + low) + floor_of(scores.dtype))
    return out


def check(name, got, want):
    """Every element of got within its bound of want = (value, bound); NaNs at the same places."""
    value, bound = want
    got = got.detach().cpu().double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    nan = torch.isnan(value)
    assert torch.equal(torch.isnan(got), nan), name
    over = torch.where(nan, torch.zeros_like(bound), (got - value).abs() - bound)
    if over.numel():
        worst = int(over.argmax())
        at = tuple(int(v) for v in torch.unravel_index(torch.tensor(worst), over.shape))
        assert float(over.flatten()[worst]) <= 0, \
            f"{name}{at}: got {float(got[at])}, expected {float(value[at])} +- {float(bound[at])}"
