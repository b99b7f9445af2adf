"""Tokens to their experts and back, and the experts' products, on what a worker holds.

A worker holds a window of the experts, as it holds rows of a vocabulary in DistributedEmbedding's ``vocab_shard``; choices of others' experts are
left out, so that the workers' results add up to those of all experts.  The reference has no counterpart.
float32, bfloat16 and float16, forward and backward (e4m3 rows: forward); sums are float32, in one order, and results are rounded once.
"""

import numbers

import torch

from .. import _lib
from .. import hip_ops
from ..utilities.slicing import compute_subshape
from ..utilities.slicing import compute_start_index
from .module import Module


class ExpertPlan:
    """The order of the choices of one batch of tokens by the experts that a worker holds.

    ``place`` int32 [tokens, chosen]: the sorted row of each choice; those of other workers' experts have places behind all that are held.
    ``offsets`` int32 [experts held + 1]: expert e's rows are ``offsets[e]`` to ``offsets[e + 1]``.  Both stay on the device."""

    __slots__ = ("place", "offsets", "window")

    def __init__(self, place, offsets, window):
        self.place, self.offsets, self.window = place, offsets, window


def _window(window, num_experts):
    low, high = (0, num_experts) if window is None else (int(w) for w in window)
    if not 0 <= low <= high <= num_experts:
        raise ValueError(f"window {(low, high)} is not inside [0, {num_experts}]")
    return low, high


def expert_plan(experts, num_experts, *, window=None):
    """The ``ExpertPlan`` of ``experts``, int32 or int64 [tokens, chosen]: the experts that each token goes to.  ``window``: ``(low, high)``, those held here (None: all).
    Choices outside it, and numbers that name no expert (-1 for a padded token), are left out.  Choices of one expert keep their order.  Up to 2047 experts held."""
    if not isinstance(num_experts, numbers.Integral) or num_experts < 0:
        raise ValueError(f"num_experts {num_experts!r} is no number of experts")
    low, high = _window(window, int(num_experts))
    if experts.dim() != 2 or experts.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"expert_plan: need int32 or int64 [tokens, chosen], got {tuple(experts.shape)} {experts.dtype}")
    res = _lib.front().expert_plan(experts, low, high)
    if res is None:
        res = _ExpertPlan.apply(experts, low, high)
    return ExpertPlan(*res, (low, high))


class _ExpertPlan(torch.autograd.Function):
    """For a trace to hold the call, as the other functions without a gradient here."""

    @staticmethod
    def forward(ctx, ids, low, high):
        res = hip_ops.expert_plan(ids, low, high)
        ctx.mark_non_differentiable(*res)
        return res


class _ExpertSortEight(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, place, offsets, scales):
        res = hip_ops.expert_sort(x, place, offsets, scales)
        ctx.mark_non_differentiable(*res)
        return res


class _ExpertLinearEight(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, offsets, x_scales, weight_scales, dtype):
        y = hip_ops.expert_linear(x, weight, offsets, x_scales, weight_scales, dtype)
        ctx.mark_non_differentiable(y)
        return y


class _ExpertSort(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, place, offsets):
        ctx.save_for_backward(place, offsets)
        ctx.dtype = x.dtype
        return hip_ops.expert_sort(x, place, offsets)[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        place, offsets = ctx.saved_tensors
        return hip_ops.expert_combine(grad if grad.dtype == ctx.dtype else grad.to(ctx.dtype), place, offsets), None, None


class _ExpertCombine(torch.autograd.Function):

    @staticmethod
    def forward(ctx, y, weights, place, offsets):
        ctx.save_for_backward(y if weights is not None and ctx.needs_input_grad[1] else None, weights, place, offsets)
        ctx.dtype = y.dtype
        return hip_ops.expert_combine(y, place, offsets, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        y, weights, place, offsets = ctx.saved_tensors
        need_y, need_w = ctx.needs_input_grad[:2]
        grad = grad if grad.dtype == ctx.dtype else grad.to(ctx.dtype)
        return _general_combine_backward(grad, y, weights, place, offsets, need_y, need_w) + (None, None)


def _general_sort_backward(grad, place, offsets):
    """The adjoint for what its native form does not take; so the others."""
    return hip_ops.expert_combine(grad, place, offsets)


def _general_combine_backward(grad, y, weights, place, offsets, want_rows, want_weights):
    if weights is None:
        return hip_ops.expert_sort(grad, place, offsets)[0] if want_rows else None, None
    return hip_ops.expert_combine_backward(grad, y, place, offsets, weights, want_rows, want_weights)


def expert_sort(x, plan, scales=None):
    """Rows ``x`` [tokens, cols] in the order of their experts, a row for each choice: [tokens * chosen, cols], zeros behind the last expert's (``plan.offsets[-1]``).

    With ``scales`` (float32, one for each token) x is moved as it is, elements of 1, 2 or 4 bytes, and ``(rows, their scales)`` is returned: rows in 8 bits, as
    ``rms_norm_shard`` and ``quantize_rows`` make them.  These have no gradient."""
    if scales is not None:
        if torch.is_grad_enabled() and (x.requires_grad or scales.requires_grad):
            raise ValueError("rows with scales have no gradient: call this under torch.no_grad(), or detach the operands")
        res = _lib.front().expert_sort_eight(x, plan.place, plan.offsets, scales)
        return res if res is not None else _ExpertSortEight.apply(x, plan.place, plan.offsets, scales)
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise ValueError(f"expert_sort: float32, bfloat16 and float16 rows, others with their scales, got {x.dtype}")
    res = _lib.front().expert_sort_shard(x, plan.place, plan.offsets, _lib.callback(_general_sort_backward))
    return res if res is not None else _ExpertSort.apply(x, plan.place, plan.offsets)


def expert_combine(y, plan, weights=None):
    """What came of each token's choices, ``y`` [tokens * chosen, cols] in the experts' order, times ``weights`` (float32 [tokens, chosen]; None: ones), added up: [tokens, cols].
    Choices that the plan left out add nothing; what lies behind the last expert's rows is not read."""
    res = _lib.front().expert_combine_shard(y, weights, plan.place, plan.offsets, _lib.callback(_general_combine_backward))
    return res if res is not None else _ExpertCombine.apply(y, weights, plan.place, plan.offsets)


class _ExpertLinear(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x, weight, offsets):
        ctx.save_for_backward(x, weight, offsets)
        return hip_ops.expert_linear(x, weight, offsets)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, offsets = ctx.saved_tensors
        grad = grad if grad.dtype == x.dtype else grad.to(x.dtype)
        return hip_ops.expert_linear_backward(grad, x, weight, offsets, *ctx.needs_input_grad[:2]) + (None,)


def _general_linear_backward(grad, x, weight, offsets, want_input, want_weight):
    return hip_ops.expert_linear_backward(grad, x, weight, offsets, want_input, want_weight)


def expert_linear_shard(x, weight, offsets, *, x_scales=None, weight_scales=None, dtype=None):
    """Rows of ``x`` [rows, in], sorted by expert, times their experts' weights [experts, out, in]: [rows, out].

    ``offsets``: int32 [experts + 1] on the device, as ``ExpertPlan.offsets``, or a part of those for a part of the experts; rows in front of the first expert's and
    behind the last one's become zeros, and take zero gradients.
    e4m3 rows (torch.float8_e4m3fn) come with ``x_scales`` [rows] and ``weight_scales`` [experts, out], both float32, and the result is in
    ``dtype`` (default bfloat16); they have no gradient, and their products are added as the matrix cores do, in eights whose members are cut off at 2^-13 of the largest.  16-bit matrices have at least 8 rows and columns, those of e4m3 a multiple of 16 columns."""
    if x.dtype == torch.float8_e4m3fn:
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x_scales, weight_scales)):
            raise ValueError("products of rows in 8 bits have no gradient: call this under torch.no_grad(), or detach the scales")
        res = None
        if x_scales is not None and weight_scales is not None:
            res = _lib.front().expert_linear_eight(x, weight, offsets, x_scales, weight_scales, torch.bfloat16 if dtype is None else dtype)
        return res if res is not None else _ExpertLinearEight.apply(x, weight, offsets, x_scales, weight_scales, dtype)
    if x_scales is not None or weight_scales is not None or dtype not in (None, x.dtype):
        raise ValueError(f"expert_linear_shard: scales and another type of the result are for e4m3 rows, these are {x.dtype}")
    res = _lib.front().expert_linear_shard(x, weight, offsets, _lib.callback(_general_linear_backward))
    return res if res is not None else _ExpertLinear.apply(x, weight, offsets)


class DistributedExpertLinear(Module):
    r"""A matrix for each of ``num_experts`` experts, which are dealt to the workers along the first dimension of ``P_x``.

    Parameters
    ----------
    P_x :
        Partition of the experts (first dimension; the others whole).
    num_experts, in_features, out_features :
        Global; a worker holds ``weight`` [its experts, out_features, in_features].  ``window`` names its experts, as ``expert_plan`` takes them.
    device, dtype :
        Of the weight.

    ``forward(x, plan)``: rows in the order of the worker's experts, as ``expert_sort`` gives them, by ``expert_linear_shard``.
    """

    def __init__(self, P_x, num_experts, in_features, out_features, device=None, dtype=None):
        super().__init__()
        self.P_x = P_x
        if not self.P_x.active:
            return
        if any(int(n) != 1 for n in P_x.shape[1:]):
            raise ValueError(f"experts are partitioned along the first dimension, got a partition of shape {list(P_x.shape)}")
        self.num_experts, self.in_features, self.out_features = int(num_experts), int(in_features), int(out_features)
        low = int(compute_start_index(P_x.shape[:1], P_x.index[:1], [self.num_experts])[0])
        self.window = (low, low + int(compute_subshape(P_x.shape[:1], P_x.index[:1], [self.num_experts])[0]))
        device = P_x.device if device is None else device
        self.weight = torch.nn.Parameter(torch.empty((self.window[1] - low, self.out_features, self.in_features), device=device, dtype=dtype))
        self.reset_parameters()

    def reset_parameters(self):
        if self.P_x.active:
            bound = self.in_features ** -0.5      # as torch.nn.Linear's
            torch.nn.init.uniform_(self.weight, -bound, bound)

    def extra_repr(self) -> str:
        return f'num_experts={self.num_experts}, in_features={self.in_features}, out_features={self.out_features}, window={self.window}' if self.P_x.active else ''

    def forward(self, x, plan):
        if not self.P_x.active:
            return x
        if plan.window != self.window:
            raise ValueError(f"the plan is of experts {plan.window}, this worker holds {self.window}")
        return expert_linear_shard(x, self.weight, plan.offsets)
