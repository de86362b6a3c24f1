"""Linear layers on MI355X: a matrix product with bias, activation and residual in one launch, and its gradients.

``linear`` has one weight matrix, as the layers of PCCSNet's classifier and synthesizer do (PCCSNet/models/components.py);
``modality_linear`` has one per modality, over rows sorted by modality (``pccs_accel.routing.sort_pairs``).

    z = x weight^T + bias,   y = activation(z) + residual

Types float32, bfloat16, float16, all tensors of a call alike; sums are float32, y is rounded once.  For the backward pass of an
activation z is kept in the same type (rounded once), and z's gradient is rounded to it for the products with weight and x; the bias'
gradient is summed before that.  Second derivatives are not offered.  All calls enqueue on the current stream, wait for nothing and
can be captured into a graph (a backward pass together with its forward pass, see ``routing``); sums have a fixed order.
"""
import torch

from . import kernels as K
from ._lib import binding


def _run(x, weight, bias, activation, residual, offsets):
    try:
        return binding().linear(x, weight, bias, K._ACT_CODE[activation], residual, offsets)
    except (TypeError, KeyError):  # not even the right kinds of objects, or no such activation
        return None


def _refuse(x, weight, bias, activation, residual, offsets):
    """The front end says what is wrong; it has no autograd node, so its result is not used."""
    K.linear(x, weight, bias, activation, residual, offsets)
    raise TypeError("linear: arguments of another kind than described")


def linear(x, weight, bias=None, activation=None, residual=None):
    """activation(x weight^T + bias) + residual.

    x [..., in] (a matrix may be a slice of columns of a larger one), weight [out, in], bias [out], residual [..., out];
    activation None, 'relu', 'gelu' (erf) or 'silu'.  Returns [..., out] in x's type."""
    y = _run(x, weight, bias, activation, residual, None)  # matrices
    if y is not None:
        return y
    if isinstance(x, torch.Tensor) and x.dim() != 2:
        if x.dim() < 1:
            raise ValueError("x: expected at least one dimension")
        lead = x.shape[:-1]
        if not x.is_contiguous() or (isinstance(residual, torch.Tensor) and not residual.is_contiguous()):
            raise ValueError("x, residual: must be contiguous unless they are matrices")
        if isinstance(residual, torch.Tensor):
            if residual.shape[:-1] != lead:
                raise ValueError(f"residual: expected {tuple(lead)} rows, got shape {tuple(residual.shape)}")
            residual = residual.reshape(lead.numel(), residual.shape[-1])
        x = x.reshape(lead.numel(), x.shape[-1])
        y = _run(x, weight, bias, activation, residual, None)
        if y is not None:
            return y.reshape(lead + (weight.shape[0],))
    return _refuse(x, weight, bias, activation, residual, None)


def modality_linear(rows, offsets, weight, bias=None, activation=None, residual=None):
    """The same with one weight matrix per modality: rows offsets[e] to offsets[e + 1] of rows [R, in] use weight[e].

    offsets int32 [E + 1] on the device, not decreasing, from 0 to at most R (``PairPlan.offsets``); weight [E, out, in],
    bias [E, out], residual [R, out].  Rows behind offsets[E] give zeros and have no gradient."""
    if offsets is None:
        raise TypeError("offsets: expected a torch.Tensor, got None")
    y = _run(rows, weight, bias, activation, residual, offsets)
    return y if y is not None else _refuse(rows, weight, bias, activation, residual, offsets)
