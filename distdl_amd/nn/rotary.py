"""Positions of queries and keys as rotations, alone or behind a norm of each head, on the heads that a worker holds.

The reference shards the projections of an attention block by heads (nn/linear_ag.py:46-60: ``num_heads``, ``num_heads_kv``,
``num_vars``) and leaves what happens to the heads to its user; these layers have no counterpart there.  Heads are whole
on their worker, so nothing is exchanged but the norms' weights.  Tensors are [batch, tokens, heads, head_dim]; queries and
keys may be views of one projection's output.  float32, bfloat16 and float16, forward and backward; angles are formed in
64 bits, sums in 32, results are rounded once.
"""

import math

import torch

from .. import _lib
from .. import hip_ops
from ..utilities.slicing import worker_layout
from ..utilities.torch import zero_volume_tensor
from .broadcast import Broadcast
from .module import Module


def rotary_frequencies(rotated, base=10000.0, scaling=None, factor=1.0, original_tokens=None, slow=1.0, fast=32.0, device=None):
    """Radians for each position of the pairs of ``rotated`` elements, float64: ``base ** (-2 p / rotated)``.

    ``scaling`` stretches them for contexts ``factor`` times longer than those of training: "linear" divides all of them,
    "base" enlarges the base so that the slowest pair is divided by ``factor`` and the fastest is left, "bands" divides pairs that turn at
    most ``slow`` times in ``original_tokens`` positions, keeps those that turn ``fast`` times or more, and goes linearly
    from one to the other between them."""
    if rotated < 0 or rotated % 2:
        raise ValueError(f"rotary_frequencies: {rotated} elements do not form pairs")
    if not base > 0 or not factor > 0:
        raise ValueError(f"rotary_frequencies: base {base} and factor {factor} must be positive")
    half = rotated // 2
    pair = torch.arange(half, dtype=torch.float64)
    if scaling == "base" and half > 1:
        base = base * factor ** (half / (half - 1))
    frequencies = float(base) ** (-pair / max(half, 1))
    if scaling == "linear":
        frequencies = frequencies / factor
    elif scaling == "bands":
        if not original_tokens or not 0 <= slow < fast:
            raise ValueError(f"rotary_frequencies: bands need original_tokens and slow < fast, got {original_tokens}, {slow}, {fast}")
        turns = original_tokens * frequencies / (2 * math.pi)
        kept = ((turns - slow) / (fast - slow)).clamp(0, 1)
        frequencies = frequencies * (kept + (1 - kept) / factor)
    elif scaling not in (None, "base"):
        raise ValueError(f"rotary_frequencies: scaling {scaling!r} is none of None, 'linear', 'base', 'bands'")
    return frequencies.to(device) if device is not None else frequencies


def _as(grad, x):
    """A gradient in the type of what it is the gradient of."""
    return grad if grad is None or grad.dtype == x else grad.detach().to(x)


class _RotaryShard(torch.autograd.Function):
    """Queries and keys turned by their positions; the adjoint turns their gradients back."""

    @staticmethod
    def forward(ctx, q, k, frequencies, positions, interleaved, amplitude):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(frequencies, positions)
        ctx.how, ctx.dtype = (interleaved, amplitude), None if q is None and k is None else (q if q is not None else k).dtype
        return hip_ops.head_rotary(q, k, frequencies, positions, interleaved, amplitude)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dyq, dyk):
        frequencies, positions = ctx.saved_tensors
        dyq, dyk = (_as(dy, ctx.dtype) if need else None for dy, need in zip((dyq, dyk), ctx.needs_input_grad))
        dq = dk = None
        if dyq is not None or dyk is not None:
            dq, dk = hip_ops.head_rotary(dyq, dyk, frequencies, positions, *ctx.how, inverse=True)
        return dq, dk, None, None, None, None


class _HeadNormRotaryShard(torch.autograd.Function):
    """Heads divided by their root mean square, times their weights, then turned; and the adjoint, which forms the norms anew
    from the heads (they are read for the gradient anyway)."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, frequencies, positions, eps, interleaved, amplitude):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, q_weight, k_weight, frequencies, positions)
        ctx.how = (interleaved, amplitude, eps)
        return hip_ops.head_rotary(q, k, frequencies, positions, interleaved, amplitude, norm=True, q_weight=_row(q_weight), k_weight=_row(k_weight),
                                   eps=eps)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dyq, dyk):
        q, k, q_weight, k_weight, frequencies, positions = ctx.saved_tensors
        need, dtype = ctx.needs_input_grad, (q if q is not None else k).dtype
        dyq = _as(dyq, dtype) if need[0] or need[2] else None
        dyk = _as(dyk, dtype) if need[1] or need[3] else None
        if dyq is None and dyk is None:
            return (None,) * 9
        dq, dk, dqw, dkw = hip_ops.head_norm_rotary_backward(dyq, dyk, q, k, _row(q_weight), _row(k_weight), frequencies, positions, *ctx.how,
                                                             want_q_weight=need[2], want_k_weight=need[3])
        return (dq if need[0] else None, dk if need[1] else None, None if dqw is None else dqw.view(q_weight.shape),
                None if dkw is None else dkw.view(k_weight.shape), None, None, None, None, None)


def _general_rotary_backward(dyq, dyk, frequencies, positions, interleaved, amplitude):
    """The adjoint for what its native form does not take."""
    return hip_ops.head_rotary(dyq, dyk, frequencies, positions, interleaved, amplitude, inverse=True)


def _general_head_norm_backward(dyq, dyk, q, k, q_weight, k_weight, frequencies, positions, interleaved, amplitude, eps, want_q_weight, want_k_weight):
    dq, dk, dqw, dkw = hip_ops.head_norm_rotary_backward(dyq, dyk, q, k, _row(q_weight), _row(k_weight), frequencies, positions, interleaved, amplitude,
                                                         eps, want_q_weight, want_k_weight)
    return dq, dk, None if dqw is None else dqw.view(q_weight.shape), None if dkw is None else dkw.view(k_weight.shape)


def _row(weight):
    return None if weight is None else weight.detach().reshape(-1)


def _refuse_gradient_of(frequencies):
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise ValueError("rotary frequencies have no gradient: detach them")


def rotary_shard(q, k, frequencies, positions=None, *, interleaved=False, amplitude=1.0):
    """``(q, k)`` turned by their positions: pair p of a head by ``position * frequencies[p]``, with ``amplitude``.

    q, k: [batch, tokens, heads, head_dim] (either may be None).  A pair is the elements p and p + len(frequencies) of a head, or
    2 p and 2 p + 1 if ``interleaved``; elements behind the pairs stay.  ``positions``: integers, [tokens] or [batch, tokens];
    None counts from 0."""
    res = _lib.front().rotary_shard(q, k, frequencies, positions, interleaved, amplitude, _lib.callback(_general_rotary_backward))
    if res is not None:
        return res
    _refuse_gradient_of(frequencies)
    # (without gradients as well: a tangent is then refused, and a trace holds the call)
    return _RotaryShard.apply(q, k, frequencies, positions, bool(interleaved), float(amplitude))


def head_norm_rotary_shard(q, k, q_weight, k_weight, frequencies, positions=None, *, eps=1e-6, interleaved=False, amplitude=1.0):
    """``rotary_shard`` of heads that are divided by ``sqrt(mean of their squares + eps)`` and multiplied by their weights
    (``head_dim`` elements of the heads' type, or None) first, in the same pass."""
    res = _lib.front().head_norm_rotary_shard(q, k, q_weight, k_weight, frequencies, positions, eps, interleaved, amplitude,
                                              _lib.callback(_general_head_norm_backward))
    if res is not None:
        return res
    _refuse_gradient_of(frequencies)
    return _HeadNormRotaryShard.apply(q, k, q_weight, k_weight, frequencies, positions, float(eps), bool(interleaved), float(amplitude))


class DistributedRotary(Module):
    r"""Rotation of queries and keys by their positions, on heads partitioned by ``P_x`` (batch, tokens, heads, head_dim;
    the last one whole).

    Parameters
    ----------
    P_x :
        Partition of queries and keys.  Where it splits the tokens, ``forward`` needs the positions of the worker's own.
    head_dim, rotated :
        Elements of a head, and those of them that turn (the first ones; None: all).
    base, scaling, factor, original_tokens, slow, fast :
        See ``rotary_frequencies``.
    interleaved :
        Pairs are neighbours instead of halves.
    amplitude :
        Factor of what turns (long-context scalings come with one).
    """

    def __init__(self, P_x, head_dim, rotated=None, base=10000.0, interleaved=False, scaling=None, factor=1.0, original_tokens=None,
                 slow=1.0, fast=32.0, amplitude=1.0, device=None):
        super().__init__()
        self.P_x = P_x
        if not self.P_x.active:
            return
        if P_x.dim != 4 or int(P_x.shape[3]) != 1:
            raise ValueError(f"heads are partitioned as [batch, tokens, heads, 1], got a partition of shape {list(P_x.shape)}")
        self.head_dim, self.rotated = int(head_dim), int(head_dim if rotated is None else rotated)
        if not 0 <= self.rotated <= self.head_dim:
            raise ValueError(f"{self.rotated} elements of heads of {self.head_dim} cannot turn")
        self.interleaved, self.amplitude = bool(interleaved), float(amplitude)
        frequencies = rotary_frequencies(self.rotated, base, scaling, factor, original_tokens, slow, fast, P_x.device if device is None else device)
        # not .to()-able to another type: the angles of far positions need its 64 bits
        self._frequencies = frequencies

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        if self.P_x.active:
            moved = fn(torch.empty(0, dtype=torch.float32, device=self._frequencies.device))
            self._frequencies = self._frequencies.to(moved.device)
        return self

    def extra_repr(self) -> str:
        return f'head_dim={self.head_dim}, rotated={self.rotated}, interleaved={self.interleaved}, amplitude={self.amplitude}'

    def _check(self, q, positions):
        if q.shape[-1] != self.head_dim:
            raise ValueError(f"heads have {q.shape[-1]} elements, the layer was built for {self.head_dim}")
        if positions is None and int(self.P_x.shape[1]) > 1:
            raise ValueError("the tokens are partitioned: pass the positions of this worker's own")

    def forward(self, q, k=None, positions=None):
        if not self.P_x.active:
            return q, k
        self._check(q, positions)
        return rotary_shard(q, k, self._frequencies, positions, interleaved=self.interleaved, amplitude=self.amplitude)


class DistributedHeadNormRotary(DistributedRotary):
    r"""``DistributedRotary`` behind a norm of each head of queries and keys, in the same pass.

    The norms' weights, ``q_weight`` and ``k_weight`` of ``head_dim`` elements, live on the first worker and are broadcast, so
    that their gradients are summed over all workers' tokens and heads.  Other parameters as ``DistributedRotary``'s, which
    are given by name; ``eps``, ``elementwise_affine``, ``dtype`` and ``scale_backward`` as ``DistributedLayerNorm``'s.
    """

    def __init__(self, P_x, head_dim, eps=1e-6, elementwise_affine=True, device=None, dtype=None, scale_backward=None, **rotary):
        super().__init__(P_x, head_dim, device=device, **rotary)
        if not self.P_x.active:
            return
        self.eps, self.elementwise_affine = float(eps), elementwise_affine
        if not elementwise_affine:
            self.register_parameter('q_weight', None)
            self.register_parameter('k_weight', None)
            return
        device = P_x.device if device is None else device
        P_w_base = P_x.create_partition_inclusive(worker_layout(P_x.shape).reshape(-1)[:1].tolist())
        self.P_w = P_w_base.create_cartesian_topology_partition([1] * P_x.dim)
        P_w_base.deactivate()
        self.broadcast = Broadcast(self.P_w, P_x, scale_backward=scale_backward)
        for name in ('q_weight', 'k_weight'):
            if self.P_w.active:
                setattr(self, name, torch.nn.Parameter(torch.ones((1, 1, 1, self.head_dim), device=device, dtype=dtype)))
            else:
                self.register_buffer(name, zero_volume_tensor(device=device, requires_grad=True, dtype=dtype))

    def forward(self, q, k=None, positions=None):
        if not self.P_x.active:
            return q, k
        self._check(q, positions)
        q_weight, k_weight = self.q_weight, self.k_weight
        if self.elementwise_affine and not self.broadcast.identity:
            q_weight, k_weight = self.broadcast(q_weight), self.broadcast(k_weight)
        for w in (q_weight, k_weight):
            if w is not None and w.dtype != q.dtype:
                raise ValueError(f"DistributedHeadNormRotary weights are {w.dtype}, the heads are {q.dtype}")
        return head_norm_rotary_shard(q, k, q_weight, k_weight if k is not None else None, self._frequencies, positions, eps=self.eps,
                                      interleaved=self.interleaved, amplitude=self.amplitude)
