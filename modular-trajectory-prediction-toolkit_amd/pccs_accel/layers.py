"""Linear layers on MI355X: a matrix product with bias, activation and residual in one launch, and its gradients.

``linear`` has one weight matrix, as the layers of PCCSNet's classifier and synthesizer do (PCCSNet/models/components.py);
``modality_linear`` has one per modality, over rows sorted by modality (``pccs_accel.routing.sort_pairs``).

    z = x weight^T + bias,   y = activation(z) + residual

Types float32, bfloat16, float16, all tensors of a call alike; sums are float32, y is rounded once.  For the backward pass of an
activation z is kept in the same type (rounded once).  Second derivatives are not offered.  All calls enqueue on the current
stream, wait for nothing and can be captured into a graph; sums have a fixed order.
"""
import torch
from torch.autograd.function import once_differentiable

from . import kernels as K


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation, offsets):
        # relu's slope can be read off y where nothing was added to it
        from_y = activation == "relu" and residual is None
        y, pre = K.linear(x, weight, bias, activation, residual, offsets, want_pre=activation not in (None, "none") and not from_y)
        ctx.save_for_backward(x, weight, y if from_y else pre, offsets)
        ctx.activation = activation
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, pre, offsets = ctx.saved_tensors
        want_x, want_w, want_b, want_r = ctx.needs_input_grad[:4]
        grad = grad.contiguous()
        dx, dw, db = K.linear_backward(grad, pre, ctx.activation, x, weight, offsets, want_x, want_w, want_b, trusted=True)
        dr = None
        if want_r:  # rows behind the last set have none
            dr = grad if offsets is None else K.linear_mask_rows(grad, offsets)
        return dx, dw if want_w else None, db, dr, None, None


def _apply(x, weight, bias, activation, residual, offsets):
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (x, weight, bias, residual)):
        return _Linear.apply(x, weight, bias, residual, activation, offsets)
    return K.linear(x, weight, bias, activation, residual, offsets)[0]


def linear(x, weight, bias=None, activation=None, residual=None):
    """activation(x weight^T + bias) + residual.

    x [..., in] (a matrix may be a slice of columns of a larger one), weight [out, in], bias [out], residual [..., out];
    activation None, 'relu', 'gelu' (erf) or 'silu'.  Returns [..., out] in x's type."""
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
        return _apply(x.reshape(lead.numel(), x.shape[-1]), weight, bias, activation, residual, None).reshape(lead + (weight.shape[0],))
    return _apply(x, weight, bias, activation, residual, None)


def modality_linear(rows, offsets, weight, bias=None, activation=None, residual=None):
    """The same with one weight matrix per modality: rows offsets[e] to offsets[e + 1] of rows [R, in] use weight[e].

    offsets int32 [E + 1] on the device, not decreasing, from 0 to at most R (``PairPlan.offsets``); weight [E, out, in],
    bias [E, out], residual [R, out].  Rows behind offsets[E] give zeros and have no gradient."""
    if offsets is None:
        raise TypeError("offsets: expected a torch.Tensor, got None")
    return _apply(rows, weight, bias, activation, residual, offsets)
