"""Rows that are learned, with their gradients: what stands between a sampled minibatch and the model that trains on it.

`embedding` looks rows up by node or token id (a frontier, a random walk); `expert_order`, `dispatch` and `combine` sort rows
by expert or node type, so that every product runs over a run of rows, and bring the results back; `product` multiplies each
expert's rows with its matrix, and `dropout` drops values without storing which.  Gradients follow through
torch's autograd, in reverse mode only: they cannot be differentiated a second time, and forward-mode tangents are refused.  All
of it may be captured into a CUDA graph, where no graph of the same leaves made outside the capture may be alive (refused).  The
GPU's default context records errors.  Several threads may use these functions at once, also beside one that samples.
"""
from collections import namedtuple

import torch

from .. import ops

ExpertOrder = namedtuple("ExpertOrder", "offsets source place")


def embedding(table, ids, scale=1.0, padding_id=None, sparse=False):
    """scale * table[ids], zeros where ids == padding_id, which takes no gradient.  The table's gradient is dense, or, with
    sparse=True, a sparse tensor of the rows that occur, each once, ascending (the backward pass then waits for their number, and
    the rows keep storage for all positions of `ids`: clone a gradient that stays)."""
    ctx = ops._context_for(ids)
    return ctx.native.nn_embedding(ctx.address, table, ids, scale, padding_id, sparse)


def expert_order(expert_ids, num_experts):
    """ops.expert_order as a named tuple (offsets, source, place)."""
    return ExpertOrder(*ops.expert_order(expert_ids, num_experts))


def dispatch(x, place):
    """Row place[t, k] of the result is x[t]: the rows of an expert next to each other.  `place`: that of an expert_order, or
    the order itself."""
    place = getattr(place, "place", place)
    ctx = ops._context_for(place)
    return ctx.native.nn_dispatch(ctx.address, x, place)


def combine(rows, place, weights=None):
    """Sum over k of weights[t, k] * rows[place[t, k]], with gradients for rows and weights.  `place` as in dispatch: no row of
    two slots."""
    place = getattr(place, "place", place)
    ctx = ops._context_for(place)
    return ctx.native.nn_combine(ctx.address, rows, place, weights)


def product(rows, weights, offsets):
    """rows[r, :] @ weights[e] for the rows offsets[e] .. offsets[e + 1] of every expert e, zeros for rows of no expert, with gradients
    for rows and weights [experts, k, n].  `offsets`: that of an expert_order, or the order itself."""
    offsets = getattr(offsets, "offsets", offsets)
    ctx = ops._context_for(offsets)
    return ctx.native.nn_product(ctx.address, rows, weights, offsets)


def dropout(x, p, seed=None):
    """ops.dropout with its gradient, which makes the mask again.  A seed that is a tensor must not change before the backward pass."""
    ctx = ops._context_for(x)
    tensor = isinstance(seed, torch.Tensor)
    return ctx.native.nn_dropout(ctx.address, x, p, 0 if tensor else ops.next_seed(seed), seed if tensor else None)


__all__ = ["ExpertOrder", "embedding", "expert_order", "dispatch", "combine", "product", "dropout"]
