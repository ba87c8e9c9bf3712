"""Operators of a mixture of experts: a mixture whose K components each hold a linear map.

The gate picks a few experts for every point (:func:`route_experts`: the E-step's softmax cut to
its leading components, or a learned router's scores), the routes are grouped by expert
(:func:`group_routes`), the experts' products run over the grouped rows
(:func:`expert_products`), and a point's results are joined by its weights
(:func:`combine_experts`)::

    weights, indices = route_experts(scores, top_k=2)
    routes = group_routes(indices, K)
    y = expert_products(x, weight, routes)        # [N top_k, d_out], grouped by expert
    out = combine_experts(y, weights, routes)     # [N, d_out]

They take float32, bfloat16 or float16 CUDA tensors (weights, their gradients and the bias are float32,
indices int32), run on the current stream of the tensors' device and hold their sums in 32 bits.  Where a tensor
input requires a gradient, the functions record one; the ``*_backward`` functions are the same
gradients without autograd; a step that is captured into a CUDA graph while an eager autograd graph of the
same leaves is alive takes those (autograd then joins the eager graph's stream to the capture, which CUDA
refuses).  Every wait inside the products' kernels is bounded: one that runs out leaves incomplete results, which
the next product on that device raises a RuntimeError for; :func:`check_expert_products` tells of it at once.
Forward-mode tangents and traced, batched (``torch.func``) or wrapped tensors are refused.  The
reference has no counterpart; its E-step (``flash_gmm/csrc/binding.cpp:35-49``) gives the scores of a fitted
mixture's gate.
"""
from typing import NamedTuple

import torch

from . import _ext, _lib

__all__ = ["Routes", "route_experts", "route_experts_backward", "group_routes", "expert_products",
           "expert_products_backward", "combine_experts", "combine_experts_backward", "check_expert_products"]


class Routes(NamedTuple):
    """The N top_k routes of N points, grouped by expert (int32 CUDA tensors).

    ``order[R]``: the routes sorted by expert (route ``n * top_k + j`` is slot j of point n), those
    without an expert last; ``offsets[K + 1]``: where each expert's begin; ``position[N, top_k]``:
    each route's place in ``order``, -1 for those without an expert."""
    order: torch.Tensor
    offsets: torch.Tensor
    position: torch.Tensor


_grad_enabled = torch.is_grad_enabled
_ops = None  # the compiled module, once loaded


def _load():
    global _ops
    _ops = _ext.load()
    return _ops


def _refuse(error, routes=None, **tensors):
    """The RuntimeError for arguments that are no tensors.  The calls below look at their tensors' attributes and hand them to
    the compiled module, which checks the rest; only what that trips over is looked at here (a call that launches one
    kernel costs the host about 6 us)."""
    for name, t in tensors.items():
        if not isinstance(t, torch.Tensor):
            raise RuntimeError(f"{name} must be a torch.Tensor") from error
    if routes is not None:
        if not isinstance(routes, Routes):
            raise RuntimeError("routes must be a Routes (of group_routes)") from error
        _refuse(error, order=routes.order, offsets=routes.offsets, position=routes.position)
    raise RuntimeError(str(error)) from error


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, scores, top_k, score_func, bias, n_groups, top_groups, renormalize, scale):
        weights, indices = _ext.load().route_experts(scores, top_k, score_func, bias, n_groups, top_groups,
                                                     renormalize, scale)
        ctx.save_for_backward(scores, indices)
        ctx.args = (score_func, renormalize, scale)
        ctx.mark_non_differentiable(indices)
        ctx.set_materialize_grads(False)
        return weights, indices

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_weights, _):
        if d_weights is None:
            return (None,) * 8
        scores, indices = ctx.saved_tensors
        return (_ext.load().route_experts_backward(d_weights, scores, indices, *ctx.args),) + (None,) * 7


def route_experts(scores, top_k, score_func="softmax", bias=None, n_groups=1, top_groups=None,
                  renormalize=True, scale=1.0):
    """The ``top_k`` experts of every point and their weights -> ``(weights[N, top_k] float32,
    indices[N, top_k] int32)``, best first.

    ``scores[N, K]``; ``score_func``: ``"softmax"`` over a row, ``"sigmoid"``, or ``"given"`` (the
    scores are values already, responsibilities for example).  ``bias[K]`` (float32) is added for the
    choice only, to keep the experts' loads balanced.  With ``n_groups > 1`` the experts form equal
    consecutive groups and only the ``top_groups`` groups (default: all) with the largest sums of
    their two best biased values are chosen from.  Ties go to the lowest index; the order is decided on
    64-bit values, without bias and with all groups kept on the scores themselves.  ``renormalize`` divides a
    point's weights by their sum, ``scale`` multiplies them.

    A score of -inf or NaN is masked and +inf counts as the largest finite value; slots that no
    unmasked expert is left for hold index -1 and weight 0.  K <= 4096, top_k <= 32, n_groups <= 32.
    The weights carry a gradient to ``scores``; the choice and ``bias`` have none."""
    try:
        if scores.requires_grad and _grad_enabled():
            return _Route.apply(scores, top_k, score_func, bias, n_groups, top_groups, renormalize, scale)
        return (_ops or _load()).route_experts(scores, top_k, score_func, bias, n_groups, top_groups, renormalize, scale)
    except (AttributeError, TypeError) as error:
        _refuse(error, scores=scores, **({} if bias is None else {"bias": bias}))


def route_experts_backward(d_weights, scores, indices, score_func="softmax", renormalize=True, scale=1.0):
    """``d_scores[N, K]`` (of the scores' type) from the weights' gradient, for the ``indices`` that
    :func:`route_experts` gave with the same ``score_func``, ``renormalize`` and ``scale``."""
    try:
        return (_ops or _load()).route_experts_backward(d_weights, scores, indices, score_func, renormalize, scale)
    except TypeError as error:
        _refuse(error, d_weights=d_weights, scores=scores, indices=indices)


def group_routes(indices, K):
    """Groups the routes of ``indices[N, top_k]`` (int32) by expert -> :class:`Routes`, stable: an
    expert's routes keep their order.  Indices outside [0, K) are routes without an expert."""
    try:
        return Routes(*(_ops or _load()).group_routes(indices, K))
    except TypeError as error:
        _refuse(error, indices=indices)


class _Products(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, order, offsets, position):
        ctx.save_for_backward(x, weight, order, offsets, position)
        return _ext.load().expert_products(x, weight, order, offsets, position)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        x, weight, *plan = ctx.saved_tensors
        dx, dw = _ext.load().expert_products_backward(dy, x, weight, *plan, ctx.needs_input_grad[0],
                                                      ctx.needs_input_grad[1])
        return dx, dw, None, None, None


def expert_products(x, weight, routes):
    """``y[r] = weight[e] @ x[n]`` for every grouped row r of ``routes`` (point n, expert e) ->
    ``y[N top_k, d_out]``; rows behind ``offsets[K]`` (routes without an expert) are 0.

    ``x[N, d_in]`` and ``weight[K, d_out, d_in]`` of one type; gradients to both.  float32 operands run
    on the tensor cores as three bf16 planes (24 bits together)."""
    try:
        order, offsets, position = routes
        if (x.requires_grad or weight.requires_grad) and _grad_enabled():
            return _Products.apply(x, weight, order, offsets, position)
        return (_ops or _load()).expert_products(x, weight, order, offsets, position)
    except (AttributeError, TypeError, ValueError) as error:
        _refuse(error, routes, x=x, weight=weight)


def expert_products_backward(dy, x, weight, routes, need_dx=True, need_dweight=True):
    """``[dx, dweight]`` from ``dy[N top_k, d_out]`` (``None`` where not needed): dx sums a point's
    rows in slot order, dweight an expert's rows; both round once."""
    try:
        order, offsets, position = routes
        return list((_ops or _load()).expert_products_backward(dy, x, weight, order, offsets, position, need_dx, need_dweight))
    except (TypeError, ValueError) as error:
        _refuse(error, routes, dy=dy, x=x, weight=weight)


def check_expert_products():
    """Raises :class:`flashgmm_b200._lib.DeviceWaitError` if a product on the current device gave up a bounded wait since the
    last check or error.  Synchronises the device: for places where the host waits anyway, and after the last product of a
    program or the replay of a captured one, which no later call looks at."""
    _lib.check_device_error(_lib.KERNELS_EXPERTS)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, order, offsets, position):
        ctx.save_for_backward(y, weights, order, offsets, position)
        return _ext.load().combine_experts(y, weights, order, offsets, position)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        dy, dw = _ext.load().combine_experts_backward(d_out, *ctx.saved_tensors)
        return dy if ctx.needs_input_grad[0] else None, dw if ctx.needs_input_grad[1] else None, None, None, None


def combine_experts(y, weights, routes):
    """``out[n] = sum_j weights[n, j] y[position[n, j]]`` -> ``out[N, d]``, slots without an expert
    left out.  ``y[N top_k, d]`` as :func:`expert_products` gives it, ``weights[N, top_k]`` float32;
    gradients to both."""
    try:
        order, offsets, position = routes
        if (y.requires_grad or weights.requires_grad) and _grad_enabled():
            return _Combine.apply(y, weights, order, offsets, position)
        return (_ops or _load()).combine_experts(y, weights, order, offsets, position)
    except (AttributeError, TypeError, ValueError) as error:
        _refuse(error, routes, y=y, weights=weights)


def combine_experts_backward(d_out, y, weights, routes):
    """``[dy, d_weights]`` from ``d_out[N, d]``; rows and slots of no expert get 0."""
    try:
        order, offsets, position = routes
        return list((_ops or _load()).combine_experts_backward(d_out, y, weights, order, offsets, position))
    except (TypeError, ValueError) as error:
        _refuse(error, routes, d_out=d_out, y=y, weights=weights)
