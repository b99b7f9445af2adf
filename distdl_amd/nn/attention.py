"""Attention on the heads that a worker holds: queries to the keys and values of an encoder's states, of a cache, or of the sequence itself.

The reference shards the projections around it by heads (nn/linear_ag.py:46-60: ``num_heads``, ``num_heads_kv``, ``num_vars``) and
leaves the attention to its user; these have no counterpart there.  Heads are whole on their worker, so nothing is exchanged.
float32, bfloat16 and float16, forward and backward; scores, softmax statistics and sums are float32.
"""

import torch

from .. import _lib
from .. import hip_ops
from .module import Module


class _AttentionShard(torch.autograd.Function):
    """Attention and its adjoint; kept for it are the operands, the result with what its rounding took (16-bit types), and one sum for each
    query and head (nothing where no adjoint follows: ``keep``)."""

    @staticmethod
    def forward(ctx, q, k, v, lengths, causal, scale, keep=True):
        if not keep:
            return hip_ops.attention(q, k, v, lengths, causal, scale)
        out, lse, rest = hip_ops.attention(q, k, v, lengths, causal, scale, want_lse=True)
        ctx.save_for_backward(q, k, v, out, lse, lengths, rest)
        ctx.how = (causal, scale)
        return out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output):
        q, k, v, out, lse, lengths, rest = ctx.saved_tensors
        if grad_output.dtype != q.dtype:
            grad_output = grad_output.detach().to(q.dtype)
        return hip_ops.attention_backward(grad_output, q, k, v, out, lse, lengths, *ctx.how, *ctx.needs_input_grad[:3], rest) + (None,) * 4


def _general_backward(grad_output, q, k, v, out, rest, lse, lengths, causal, scale, want_q, want_k, want_v):
    """The adjoint for what its native form does not take.  ``q``, ``k``, ``v``, ``out`` and ``rest`` may be copies whose heads are padded with zeros."""
    own = grad_output.shape[-1]
    q, k, v, out, rest = (None if t is None else t[..., :own] for t in (q, k, v, out, rest))
    return hip_ops.attention_backward(grad_output, q, k, v, out, lse, lengths, causal, scale, want_q, want_k, want_v, rest)


def attention_shard(q, k, v, lengths=None, *, causal=False, scale=None):
    """``softmax(scale q k^T) v`` for each head.

    q: [batch, tokens, heads, head_dim]; k, v: [batch, keys, kv_heads, head_dim], ``heads`` a multiple of ``kv_heads`` (head h
    uses key head ``h * kv_heads // heads``), head_dim up to 128.  ``lengths``: int32 [batch], the keys that each sequence has
    (None: all); what lies behind them is not read and gets zero gradients.  ``causal``: query i sees keys up to
    ``i + keys - tokens``, so the last query sees all.  A query that sees no key gives zeros.  ``scale`` defaults to
    ``head_dim ** -0.5`` and has to be positive."""
    out = _lib.front().attention_shard(q, k, v, lengths, causal, scale, _lib.callback(_general_backward))
    if out is not None:
        return out
    # (through the function without gradients as well: a tangent is then refused, and a trace holds the call)
    keep = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return _AttentionShard.apply(q, k, v, lengths, bool(causal), scale, keep)


class DistributedAttention(Module):
    r"""Attention of queries to keys and values whose heads (and batch) are partitioned by ``P_x`` (batch, tokens, heads,
    head_dim; tokens and head_dim whole): every worker attends with its own heads.

    Parameters
    ----------
    P_x :
        Partition of queries, keys and values.
    causal, scale :
        See ``attention_shard``.
    """

    def __init__(self, P_x, causal=False, scale=None):
        super().__init__()
        self.P_x = P_x
        if not self.P_x.active:
            return
        if P_x.dim != 4 or int(P_x.shape[1]) != 1 or int(P_x.shape[3]) != 1:
            raise ValueError(f"attention needs whole sequences and heads, [batch, 1, heads, 1], got a partition of shape {list(P_x.shape)}")
        if scale is not None and not scale > 0:
            raise ValueError(f"scale {scale} is not positive")
        self.causal, self.scale = bool(causal), scale

    def extra_repr(self) -> str:
        return f'causal={self.causal}, scale={self.scale}' if self.P_x.active else ''

    def forward(self, q, k, v, lengths=None):
        if not self.P_x.active:
            return q
        return attention_shard(q, k, v, lengths, causal=self.causal, scale=self.scale)
