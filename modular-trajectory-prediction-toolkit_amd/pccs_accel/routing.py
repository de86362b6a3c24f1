"""Routing of agents to modalities on MI355X, with gradients.

Between the classifier's scores and the candidates PCCSNet takes each agent's k most probable modalities and runs the
following layers once per (agent, modality) pair (PCCSNet/models/components.py:116-131).  Here: the k modalities with their
weights (``route_topk``), the pairs sorted by modality (``sort_pairs``), the agents' rows copied to their pairs
(``dispatch``) and the pairs' answers summed back per agent (``combine``).  ``pccs_accel.layers.modality_linear`` is the
layer with one weight matrix per modality that runs over the sorted rows.

Types float32, bfloat16, float16; softmax statistics, weights and sums are float32.  Gradients go to the scores, the rows
and the weights; second derivatives are not offered.  All calls enqueue on the current stream, wait for nothing and can be
captured into a graph; sums have a fixed order.  A backward pass is captured with its forward pass: a call under capture whose
inputs belong to a graph of autograd that was begun outside (a leaf that an eager result still refers to) is refused, since its
backward pass would end the process.  Refused as well: tracing, which does not see the kernels, forward mode, and views with the negative
bit.
"""
from typing import NamedTuple

import torch

from . import kernels as K
from ._lib import binding


def _refuse(name, explain, *args):
    """Where the arguments are not as they have to be, the front end in ``kernels`` says what is wrong; it has no autograd node, so
    its result is not used."""
    explain(*args)
    raise TypeError(f"{name}: arguments of another kind than described")


def _explain_sort(ids, n_modalities):
    if isinstance(ids, torch.Tensor) and ids.dim() != 2:
        raise ValueError(f"ids: expected [N, k], got shape {tuple(ids.shape)}")
    K.sort_pairs(ids, n_modalities)


class PairPlan(NamedTuple):
    """The (agent, modality) pairs sorted by modality; all tensors int32 on the device.

    offsets [E + 1]: modality e has the rows offsets[e] to offsets[e + 1]; pairs without a modality (id outside [0, E)) are
    behind offsets[E].  order [N * k]: the pair (agent * k + choice) of each row.  position [N, k]: the row of each pair; one
    outside [0, N * k), which no sort gives, is left out."""
    offsets: torch.Tensor
    order: torch.Tensor
    position: torch.Tensor


def route_topk(scores, k, normalize=True):
    """(ids int32 [N, k], weights float32 [N, k]): the k largest scores of each row, largest first, equal ones by the lower
    index, and their softmax weights -- over the chosen k (``normalize=True``) or over all E modalities.

    scores [N, E], E <= 4096, k <= min(E, 128).  A score of -inf forbids the modality: where fewer than k are left, ids are -1
    and weights 0.  A NaN is never chosen before another score and makes its row's weights NaN."""
    try:
        got = binding().route_topk(scores, k, bool(normalize))
    except TypeError:  # not even the right kinds of objects
        got = None
    return got if got is not None else _refuse("route_topk", K.route_topk, scores, k, normalize)


def sort_pairs(ids, n_modalities):
    """The pairs of ids int32 [N, k] sorted by modality (stable): a ``PairPlan``.  n_modalities <= 4096."""
    try:
        got = binding().sort_pairs(ids, n_modalities)
    except TypeError:
        got = None
    return PairPlan(*got) if got is not None else _refuse("sort_pairs", _explain_sort, ids, n_modalities)


def dispatch(x, plan):
    """rows [N * k, D]: agent t's row of x [N, D] at each of its pairs' places; zeros behind the last modality's rows."""
    try:
        got = binding().dispatch(x, plan.position, plan.offsets)
    except TypeError:
        got = None
    return got if got is not None else _refuse("dispatch", K.dispatch_rows, x, plan.position, plan.offsets)


def combine(rows, plan, weights=None):
    """[N, D]: for each agent the sum of its pairs' rows [N * k, D], times weights float32 [N, k] if given.  Pairs without a
    modality are left out."""
    try:
        got = binding().combine(rows, plan.position, plan.offsets, weights)
    except TypeError:
        got = None
    return got if got is not None else _refuse("combine", K.combine_rows, rows, plan.position, plan.offsets, weights)
