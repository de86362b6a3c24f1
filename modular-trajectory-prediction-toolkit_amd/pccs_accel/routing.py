"""Routing of agents to modalities on MI355X, with gradients.

Between the classifier's scores and the candidates PCCSNet takes each agent's k most probable modalities and runs the
following layers once per (agent, modality) pair (PCCSNet/models/components.py:116-131).  Here: the k modalities with their
weights (``route_topk``), the pairs sorted by modality (``sort_pairs``), the agents' rows copied to their pairs
(``dispatch``) and the pairs' answers summed back per agent (``combine``).  ``pccs_accel.layers.modality_linear`` is the
layer with one weight matrix per modality that runs over the sorted rows.

Types float32, bfloat16, float16; softmax statistics, weights and sums are float32.  Gradients go to the scores, the rows
and the weights; second derivatives are not offered.  All calls enqueue on the current stream, wait for nothing and can be
captured into a graph; sums have a fixed order.
"""
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from . import kernels as K


class PairPlan(NamedTuple):
    """The (agent, modality) pairs sorted by modality; all tensors int32 on the device.

    offsets [E + 1]: modality e has the rows offsets[e] to offsets[e + 1]; pairs without a modality (id outside [0, E)) are
    behind offsets[E].  order [N * k]: the pair (agent * k + choice) of each row.  position [N, k]: the row of each pair."""
    offsets: torch.Tensor
    order: torch.Tensor
    position: torch.Tensor


class _RouteTopk(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, k, normalize):
        ids, weights, stats = K.route_topk(scores, k, normalize, want_stats=True)
        ctx.save_for_backward(scores, ids, weights, stats)
        ctx.normalize = normalize
        ctx.mark_non_differentiable(ids)
        ctx.set_materialize_grads(False)
        return ids, weights

    @staticmethod
    @once_differentiable
    def backward(ctx, _, grad):
        if grad is None:
            return None, None, None
        scores, ids, weights, stats = ctx.saved_tensors
        return K.route_topk_grad(scores, ids, weights, stats, grad.contiguous(), ctx.normalize, trusted=True), None, None


def route_topk(scores, k, normalize=True):
    """(ids int32 [N, k], weights float32 [N, k]): the k largest scores of each row, largest first, equal ones by the lower
    index, and their softmax weights -- over the chosen k (``normalize=True``) or over all E modalities.

    scores [N, E], E <= 4096, k <= min(E, 128).  A score of -inf forbids the modality: where fewer than k are left, ids are -1
    and weights 0.  A NaN is never chosen before another score and makes its row's weights NaN."""
    if torch.is_grad_enabled() and isinstance(scores, torch.Tensor) and scores.requires_grad:
        return _RouteTopk.apply(scores, k, bool(normalize))
    return K.route_topk(scores, k, normalize)[:2]


def sort_pairs(ids, n_modalities):
    """The pairs of ids int32 [N, k] sorted by modality (stable): a ``PairPlan``.  n_modalities <= 4096."""
    if isinstance(ids, torch.Tensor) and ids.dim() != 2:
        raise ValueError(f"ids: expected [N, k], got shape {tuple(ids.shape)}")
    return PairPlan(*K.sort_pairs(ids, n_modalities))


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, position, offsets):
        ctx.save_for_backward(position, offsets)
        return K.dispatch_rows(x, position, offsets)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        return K.combine_rows(grad.contiguous(), *ctx.saved_tensors, trusted=True), None, None


def dispatch(x, plan):
    """rows [N * k, D]: agent t's row of x [N, D] at each of its pairs' places; zeros behind the last modality's rows."""
    if torch.is_grad_enabled() and isinstance(x, torch.Tensor) and x.requires_grad:
        return _Dispatch.apply(x, plan.position, plan.offsets)
    return K.dispatch_rows(x, plan.position, plan.offsets)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, position, offsets):
        y = K.combine_rows(rows, position, offsets, weights)
        # the rows themselves are needed for the weights' gradient only
        ctx.has_weights = weights is not None
        ctx.save_for_backward(rows if ctx.has_weights else None, weights, position, offsets)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        rows, weights, position, offsets = ctx.saved_tensors
        grad = grad.contiguous()
        if not ctx.has_weights:
            return K.dispatch_rows(grad, position, offsets, trusted=True), None, None, None
        want_rows, want_weights = ctx.needs_input_grad[:2]
        return K.combine_rows_grad(rows, grad, position, offsets, weights, want_rows, want_weights,
                                   trusted=True) + (None, None)


def combine(rows, plan, weights=None):
    """[N, D]: for each agent the sum of its pairs' rows [N * k, D], times weights float32 [N, k] if given.  Pairs without a
    modality are left out."""
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (rows, weights)):
        return _Combine.apply(rows, weights, plan.position, plan.offsets)
    return K.combine_rows(rows, plan.position, plan.offsets, weights)
