"""`route_experts`, which chooses each token's experts and lays out the plan that `grouped_linear` reads, and `combine_experts`, which brings the
experts' rows back to their tokens.  Neither has a counterpart in the reference.  Inference only, as every operator here."""
from __future__ import annotations

from operator import index

import torch

from .. import _rocm_ops


def route_experts(logits, top_k, scoring="softmax", bias=None, groups=1, top_groups=None, group_best=1, renormalize=True, scale=1.0):
    """Each token's top_k experts by router logits [.., E] (bf16, fp16 or fp32, E up to 1024, top_k up to 64), and the plan of the linears behind.

    The score of an expert is the softmax over all E logits, or with scoring="sigmoid" 1 / (1 + exp(-logit)); its key is the score plus bias
    (fp32 [E], for balance), both in 64 bits; without a bias (and with group_best=1) the logits themselves are compared, whose order is the same.  A token
    takes the experts of the largest keys, ties to the lowest index.  With top_groups, E is cut into `groups` equal
    ranges, and only experts of those top_groups ranges are taken whose group_best (1 or 2) largest keys have the largest sum.  Its weights are the
    scores, without the bias, over their sum with renormalize, times scale.
    An expert with a logit of -inf is not taken: a token with fewer than top_k others has expert -1, weight 0 and place -1 in its last slots, a
    row of -inf (padding) in all.  A NaN counts as the largest key, and a row with one has NaN among its weights.

    Returns (weights fp32 [.., top_k], experts int32 [.., top_k], offsets int32 [E+1], rows int32 [tokens * top_k], places int32 [.., top_k]):
    expert e has the rows from offsets[e] to offsets[e+1], the tokens in rising order; rows holds the token of each (-1 behind the last one), places the
    row of each slot.  `grouped_linear(x, .., offsets, rows)` takes tokens to their experts, `combine_experts(y, weights, places)` back.  The call does not wait for the GPU.
    """
    if not isinstance(logits, torch.Tensor) or logits.dim() < 1:
        raise RuntimeError("logits must be a tensor of at least one dim")
    view = _rocm_ops._rows_view(logits, "logits")
    if view is None:
        logits = logits.contiguous()
        view = _rocm_ops._rows_view(logits, "logits")
    try:
        top_k, groups, group_best = index(top_k), index(groups), index(group_best)
        top_groups = groups if top_groups is None else index(top_groups)
    except TypeError:
        raise RuntimeError("top_k, groups, top_groups and group_best must be whole numbers") from None
    return _rocm_ops.route_experts(logits, top_k, bias, scoring, groups, top_groups, group_best, renormalize, float(scale), view)


def combine_experts(y, weights, places, residual=None, out=None):
    """out[t] = residual[t] + sum over s of weights[t, s] * y[places[t, s]]: the experts' rows back to their tokens.

    y [M, N] in bf16, fp16 or fp32, as `grouped_linear` returns it; weights fp32 and places int32 [.., k], as `route_experts` returns them; residual
    [.., N] of y's type.  The sum is in 32 bits, in the order of the slots, rounded once.  A place of -1, or behind the last row, adds nothing.
    Returns [.., N] in y's type, into `out`, which may be residual itself.
    """
    if not isinstance(y, torch.Tensor) or y.dim() != 2 or not isinstance(places, torch.Tensor) or places.dim() < 1:
        raise RuntimeError("y must be a 2d matrix and places [.., k]")
    if not y.is_contiguous() and _rocm_ops._rows_view(y, "y") is None:
        y = y.contiguous()
    if isinstance(residual, torch.Tensor) and not residual.is_contiguous() and _rocm_ops._rows_view(residual, "residual") is None:
        if out is residual:
            raise RuntimeError("out must have rows of contiguous elements, evenly apart")
        residual = residual.contiguous()
    return _rocm_ops.combine_experts(out, y, weights, places, residual)
