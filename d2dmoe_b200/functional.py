"""Differentiable operators in front of the layer: its norm, and routing with weights.

Both run as autograd functions over the CUDA library (``ops.layer_norm`` / ``ops.route`` and their backward
passes); without a gradient to compute they are the plain calls.  First derivatives only.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import ops


def _wants_grad(*ts) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in ts)


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, kind, weight_offset):
        y, mean, rstd = ops.layer_norm(x, weight, bias, eps, kind=kind, weight_offset=weight_offset)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.how = dict(kind=kind, weight_offset=weight_offset)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, mean, rstd = ctx.saved_tensors
        want = ctx.needs_input_grad
        dx, dw, db = ops.layer_norm_backward(dy, x, weight, mean, rstd, dx=want[0], dweight=want[1],
                                             bias=want[2], **ctx.how)
        return dx, dw, db, None, None, None


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, kind="layer", weight_offset=0.0):
    """Norm of the rows of x [.., d] as the upstream blocks have it in front of the layer
    (architectures/moe/moe_models.py:69-76, :91-100, :148-156), differentiable in x, weight and bias.

    ``kind`` 'layer': (x - mean) / sqrt(var + eps) * (weight + weight_offset) + bias; 'rms': the same with a mean of
    zero (weight_offset 1 is the Gemma form).  fp32 or bf16, parameters in fp32 or x's dtype; fp32
    statistics, one rounding.  The parameters' gradients are summed over all rows in fp32 and in a fixed order."""
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, eps, kind, weight_offset)
    return ops.layer_norm(x, weight, bias, eps, kind=kind, weight_offset=weight_offset, statistics=False)[0]


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, how, bias, groups, top_groups):
        weights, experts, _ = ops.route(logits, k, bias=bias, groups=groups, top_groups=top_groups, **how)
        ctx.save_for_backward(logits, experts, weights)
        ctx.how = how
        ctx.set_materialize_grads(False)
        ctx.mark_non_differentiable(experts)
        return weights, experts

    @staticmethod
    @once_differentiable
    def backward(ctx, dweights, _):
        if dweights is None:
            return (None,) * 6
        logits, experts, weights = ctx.saved_tensors
        return ops.route_backward(dweights, logits, experts, weights, **ctx.how), None, None, None, None, None


def route_tokens(logits, k, *, scores="softmax", bias=None, groups=1, top_groups=None, renormalise=True,
                 scale=1.0):
    """Token-choice routing: ``(weights [.., k] fp32, experts [.., k] int32)`` of router logits [.., E], the
    weights differentiable in the logits (the choice, and the balance ``bias`` that moves it, have no gradient).

    scores 'softmax' or 'sigmoid'; experts are chosen by score + bias (fp32 [E]; not part of the weights), the best
    first, ties to the lowest index; with ``groups`` > 1 only from the ``top_groups`` groups whose two best experts sum
    highest; ``renormalise``: weights sum to ``scale`` over a token's experts.  The choice is the one that 64-bit
    arithmetic makes.  Logits of -inf are never chosen; slots left over have expert -1 and weight 0."""
    top_groups = groups if top_groups is None else top_groups
    how = dict(scores=scores, renormalise=renormalise, scale=scale)
    if _wants_grad(logits):
        return _Route.apply(logits, k, how, bias, groups, top_groups)
    return ops.route(logits, k, bias=bias, groups=groups, top_groups=top_groups, **how)[:2]
