"""Root-mean-square norm of a partitioned tensor, with the residual's addition and an 8-bit output in the same pass.

It stands beside DistributedLayerNorm (reference: nn/layernorm.py:15-321, whose constructor it follows); the reference has no counterpart.
float32, bfloat16 and float16, forward and backward; sums are float32 and results are rounded once.
"""

import numbers

import numpy as np
import torch

from .. import _lib
from .. import hip_ops
from ..utilities.slicing import compute_subshape
from ..utilities.slicing import range_index
from ..utilities.slicing import worker_layout
from ..utilities.torch import zero_volume_tensor
from .all_sum_reduce import AllSumReduce
from .broadcast import Broadcast
from .module import Module

SQUARES_TAG = "rms_norm_squares"
BWD_SUMS_TAG = "rms_norm_backward_sums"


def _gathered(P_reduce, sums, tag):
    return P_reduce._world.transport.allgather(P_reduce, sums, tag=tag).contiguous()


class _RmsNormShard(torch.autograd.Function):
    """The norm of the rows of x, or of x + residual, which it returns as well; its adjoint forms the rows' statistics anew.  Kept: the rows that
    were normalised (the second result) and, where the columns are spread over ``P_reduce``, all workers' sums of squares."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps, P_reduce, total_cols):
        ctx.set_materialize_grads(False)
        w = None if weight is None else weight.detach().reshape(-1)
        squares = None
        if P_reduce is None:
            y, h, _, _ = hip_ops.rms_norm(x, w, residual, eps)
        else:
            squares, h = hip_ops.rms_norm(x, None, residual, eps, own_squares=True)
            squares = _gathered(P_reduce, squares, SQUARES_TAG)
            y = hip_ops.rms_norm(h, w, None, eps, part_squares=squares, total_cols=total_cols)[0]
        ctx.save_for_backward(h, weight, squares)
        ctx.how = eps, P_reduce, total_cols, residual is not None
        return y if residual is None else (y, h)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, squares = ctx.saved_tensors
        eps, P_reduce, total_cols, added = ctx.how
        need_x, need_w, need_r = ctx.needs_input_grad[:3]
        dy, dh = (t if t is None or t.dtype == h.dtype else t.detach().to(h.dtype) for t in (dy, dh))
        dx = dw = None
        if dy is None:       # only the sum was used
            dx = dh
            if P_reduce is not None:    # the other workers wait for these
                _gathered(P_reduce, torch.zeros(h.numel() // h.shape[-1], dtype=torch.float32, device=h.device), BWD_SUMS_TAG)
            if need_w and weight is not None:
                dw = torch.zeros_like(weight)
        else:
            w = None if weight is None else weight.detach().reshape(-1)
            sums = None
            if P_reduce is not None:
                sums = hip_ops.rms_norm_backward(dy, h, w, None, eps, own_sums=True)
                sums = _gathered(P_reduce, sums, BWD_SUMS_TAG)
            dx, dw = hip_ops.rms_norm_backward(dy, h, w, dh, eps, need_x or need_r, need_w, part_squares=squares, part_sums=sums, total_cols=total_cols)
            if dw is not None:
                dw = dw.view(weight.shape)
        return dx if need_x else None, dw, dx if need_r else None, None, None, None


def _general_backward(dy, h, weight, dh, eps, want_input, want_weight):
    """The adjoint for what its native form does not take."""
    dx, dw = hip_ops.rms_norm_backward(dy, h, None if weight is None else weight.detach().reshape(-1), dh, eps, want_input, want_weight)
    return dx, None if dw is None else dw.view(weight.shape)


class _RmsNormEight(torch.autograd.Function):
    """Rows in 8 bits, for a trace to hold the call and a tangent to be refused."""

    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        _, h, codes, scales = hip_ops.rms_norm(x, None if weight is None else weight.detach().reshape(-1), residual, eps, eight_bit=True)
        res = (codes, scales) if residual is None else (codes, scales, h)
        ctx.mark_non_differentiable(*res)
        return res


class _QuantizeRows(torch.autograd.Function):

    @staticmethod
    def forward(ctx, x):
        res = hip_ops.quantize_rows(x)
        ctx.mark_non_differentiable(*res)
        return res


def rms_norm_shard(x, weight=None, residual=None, *, eps=1e-6, eight_bit=False):
    """Rows (the last dimension) of ``x`` divided by ``sqrt(mean of their squares + eps)`` and multiplied by ``weight`` (its elements, of x's type, or None).

    With ``residual`` (like x) the rows of ``h = x + residual``, rounded to their type, are normalised, and ``(y, h)`` is returned: h is the
    stream that goes on.  ``eight_bit``: instead of y its ``codes`` (torch.float8_e4m3fn) and ``scales`` (float32, one a row), ``code = e4m3(y / scale)``, ``scale =
    max(max |y| / 448, 2^-126)``: ``(codes, scales)`` or ``(codes, scales, h)``.  These have no gradient, so they are refused where one would be recorded.  Up to
    16384 columns.  The sum of a row's squares has to be a float32."""
    if not eight_bit:
        res = _lib.front().rms_norm_shard(x, weight, residual, eps, _lib.callback(_general_backward))
        if res is not None:
            return res[0] if residual is None else res
        return _RmsNormShard.apply(x, weight, residual, float(eps), None, None)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise ValueError("rows in 8 bits have no gradient: call this under torch.no_grad(), or detach the operands")
    res = _lib.front().rms_norm_eight(x, weight, residual, eps)
    if res is not None:
        return res[:2] if residual is None else res
    return _RmsNormEight.apply(x, weight, residual, float(eps))


def quantize_rows(x):
    """``(codes, scales)``: rows (the last dimension) of ``x`` in 8 bits, ``code = e4m3(x / scale)``, ``scale = max(max |x| / 448, 2^-126)`` for each row (by
    the rounded 1 / 448; the code is that of the rounded quotient).  A row with an infinity in it stands for no numbers.  No gradient."""
    if torch.is_grad_enabled() and x.requires_grad:
        raise ValueError("rows in 8 bits have no gradient: call this under torch.no_grad(), or detach the operand")
    res = _lib.front().quantize_rows(x)
    return res if res is not None else _QuantizeRows.apply(x)


class DistributedRMSNorm(Module):
    r"""Root-mean-square norm over the last ``len(normalized_shape)`` dimensions of a tensor partitioned by ``P_x``; those dimensions may
    themselves be partitioned.

    Parameters
    ----------
    P_x :
        Partition of the input (and output) tensor.
    normalized_shape :
        Global extent(s) of the normalised dimensions, on a worker up to 16384 elements.
    eps, elementwise_affine, device, dtype, scale_backward :
        As ``DistributedLayerNorm``'s.  There is no bias.

    ``forward(x, residual=None, eight_bit=False)`` returns what ``rms_norm_shard`` does.  Rows in 8 bits need whole rows.
    """

    def __init__(self, P_x, normalized_shape, eps=1e-6, elementwise_affine=True, device=None, dtype=None, scale_backward=None):
        super().__init__()
        self.P_x = P_x
        if not self.P_x.active:
            return
        if isinstance(normalized_shape, numbers.Integral):
            normalized_shape = (normalized_shape,)
        self.normalized_shape = tuple(int(n) for n in normalized_shape)
        self.eps, self.elementwise_affine = float(eps), elementwise_affine
        first = P_x.dim - len(self.normalized_shape)
        if first < 0:
            raise ValueError(f"{len(self.normalized_shape)} normalised dimensions of a partition of {P_x.dim}")
        self.allreduce = AllSumReduce(P_x, axes_reduce=tuple(range(first, P_x.dim)))
        reduce_shape = np.asarray(P_x.shape[first:]).astype(int)
        self.split = int(np.prod(reduce_shape)) > 1
        self.total_cols = int(np.prod(self.normalized_shape))
        local = tuple(int(n) for n in compute_subshape(reduce_shape, P_x.index[first:], self.normalized_shape))
        self.local_shape = local
        least = min(int(np.prod(compute_subshape(reduce_shape, idx, self.normalized_shape))) for idx in range_index(reduce_shape))
        if least < 1:
            raise ValueError(f"a worker has no elements of normalized_shape={self.normalized_shape}")
        if not elementwise_affine:
            self.register_parameter('weight', None)
            return
        device = P_x.device if device is None else device
        # The weight lives on the workers with index 0 in every dimension that is not normalised, and is broadcast along those.
        weight_partition_shape = np.copy(P_x.shape)
        weight_partition_shape[:first] = 1
        index = [0] * first + [slice(0, int(n)) for n in reduce_shape]
        P_w_base = P_x.create_partition_inclusive(worker_layout(P_x.shape)[tuple(index)].reshape(-1).tolist())
        self.P_w = P_w_base.create_cartesian_topology_partition(weight_partition_shape)
        P_w_base.deactivate()
        self.broadcast = Broadcast(self.P_w, P_x, scale_backward=scale_backward)
        if self.P_w.active:
            self.weight = torch.nn.Parameter(torch.ones((1,) * first + local, device=device, dtype=dtype))
        else:
            self.register_buffer('weight', zero_volume_tensor(device=device, requires_grad=True, dtype=dtype))

    def extra_repr(self) -> str:
        return f'normalized_shape={self.normalized_shape}, eps={self.eps}' if self.P_x.active else ''

    def forward(self, x, residual=None, eight_bit=False):
        if not self.P_x.active:
            return x if residual is None else (x, residual)
        dims = len(self.normalized_shape)
        if x.dim() < dims or tuple(x.shape[x.dim() - dims:]) != self.local_shape:
            raise ValueError(f"input shard {tuple(x.shape)}: the partition of normalized_shape={self.normalized_shape} gives this worker {self.local_shape}")
        if eight_bit and self.split:
            raise ValueError("rows in 8 bits have a scale each, so they have to be whole on their worker")
        weight = self.weight
        if self.elementwise_affine and not self.broadcast.identity:
            weight = self.broadcast(weight)
        if weight is not None and weight.dtype != x.dtype:
            raise ValueError(f"DistributedRMSNorm's weight is {weight.dtype}, the input is {x.dtype}")
        shape, flat = x.shape, x.shape[:x.dim() - dims] + (int(np.prod(self.local_shape)),)
        if residual is not None and residual.shape != shape:
            raise ValueError(f"residual {tuple(residual.shape)} of an input {tuple(shape)}")
        if dims > 1:
            x, residual = x.reshape(flat), None if residual is None else residual.reshape(flat)
        if self.split:
            res = _RmsNormShard.apply(x, weight, residual, self.eps, self.allreduce.P_allreduce, self.total_cols)
        else:
            res = rms_norm_shard(x, weight, residual, eps=self.eps, eight_bit=eight_bit)
        if dims == 1:
            return res
        if isinstance(res, tuple):
            return tuple(r if i == 1 and eight_bit else r.view(shape) for i, r in enumerate(res))
        return res.view(shape)
