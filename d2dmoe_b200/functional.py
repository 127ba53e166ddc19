"""Differentiable operators in front of the layer: its norm, and routing with weights.

Both run under autograd over the CUDA library (``ops.layer_norm`` / ``ops.route`` and their backward
passes, in native code); without a gradient to compute they are the plain calls.  First derivatives in reverse mode only:
a tensor with a forward-mode tangent is refused.
"""
from __future__ import annotations

import torch

from . import ops
from ._capi import host


def _wants_grad(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, kind="layer", weight_offset=0.0):
    """Norm of the rows of x [.., d] as the upstream blocks have it in front of the layer
    (architectures/moe/moe_models.py:69-76, :91-100, :148-156), differentiable in x, weight and bias.

    ``kind`` 'layer': (x - mean) / sqrt(var + eps) * (weight + weight_offset) + bias; 'rms': the same with a mean of
    zero (weight_offset 1 is the Gemma form).  fp32 or bf16, parameters in fp32 or x's dtype; fp32
    statistics, one rounding.  The parameters' gradients are summed over all rows in fp32 and in a fixed order."""
    if _wants_grad(x, weight, bias):
        return ops._refused(host.layer_norm_autograd(x, weight, bias, eps, ops.norm_kind(kind), weight_offset),
                            "d2d_layer_norm")
    return ops.layer_norm(x, weight, bias, eps, kind=kind, weight_offset=weight_offset, statistics=False)[0]


def route_tokens(logits, k, *, scores="softmax", bias=None, groups=1, top_groups=None, renormalise=True,
                 scale=1.0):
    """Token-choice routing: ``(weights [.., k] fp32, experts [.., k] int32)`` of router logits [.., E], the
    weights differentiable in the logits (the choice, and the balance ``bias`` that moves it, have no gradient).

    scores 'softmax' or 'sigmoid'; experts are chosen by score + bias (fp32 [E]; not part of the weights), the best
    first, ties to the lowest index; with ``groups`` > 1 only from the ``top_groups`` groups whose two best experts sum
    highest; ``renormalise``: weights sum to ``scale`` over a token's experts.  The choice is the one that 64-bit
    arithmetic makes.  Logits of -inf are never chosen; slots left over have expert -1 and weight 0."""
    if _wants_grad(logits):
        return ops._refused(host.route_autograd(logits, k, ops.score_kind(scores), bias, groups,
                                                groups if top_groups is None else top_groups, renormalise, scale),
                            "d2d_route")
    return ops.route(logits, k, scores=scores, bias=bias, groups=groups, top_groups=top_groups,
                     renormalise=renormalise, scale=scale)[:2]
