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


def _causal_form(causal, own_ends):
    if own_ends and not causal:
        raise ValueError("own_ends says where the causal form ends: it needs causal=True")
    return hip_ops.CAUSAL_OWN_ENDS if own_ends else int(bool(causal))


def attention_shard(q, k, v, lengths=None, *, causal=False, scale=None, own_ends=False):
    """``softmax(scale q k^T) v`` for each head.

    q: [batch, tokens, heads, head_dim]; k, v: [batch, keys, kv_heads, head_dim], ``heads`` a multiple of ``kv_heads`` (head h
    uses key head ``h * kv_heads // heads``), head_dim up to 128.  ``lengths``: int32 [batch], the keys that each sequence has
    (None: all); what lies behind them is not read and gets zero gradients.  ``causal``: query i sees keys up to
    ``i + keys - tokens``, so the last query sees all that the tensor has room for: the form for padded sequences that attend to themselves.
    With ``own_ends`` it is ``i + lengths[b] - tokens``: the queries are the last tokens of each sequence, as where several new ones
    meet a cache whose sequences have different lengths (without it the shorter sequences' first tokens would see those behind them).
    A query that sees no key gives zeros.  ``scale`` defaults to ``head_dim ** -0.5`` and has to be positive.

    Values of keys that a sequence has are to be finite, for gradients all operands, also where a query does not see a key (zero times infinity is no number).  16-bit types
    round probabilities, and dS in the adjoint, to theirs for the products.  Where gradients are recorded, 16-bit types keep a tensor as large as the
    result beside it, what its rounding took, which the adjoint needs for small differences.  Heads that are no multiple of 16 bytes, and operands that
    do not lie at multiples of 16 bytes, are copied at every call, a cache as well."""
    causal = _causal_form(causal, own_ends)
    out = _lib.front().attention_shard(q, k, v, lengths, causal, scale, _lib.callback(_general_backward))
    if out is not None:
        return out
    # (through the function without gradients as well: a tangent is then refused, and a trace holds the call)
    keep = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    return _AttentionShard.apply(q, k, v, lengths, causal, scale, keep)


class DistributedAttention(Module):
    r"""Attention of queries to keys and values whose heads (and batch) are partitioned by ``P_x`` (batch, tokens, heads,
    head_dim; tokens and head_dim whole): every worker attends with its own heads.

    Parameters
    ----------
    P_x :
        Partition of queries, keys and values.  ``lengths`` of ``forward`` are those of the worker's own sequences.
    causal, scale, own_ends :
        See ``attention_shard``.
    """

    def __init__(self, P_x, causal=False, scale=None, own_ends=False):
        super().__init__()
        self.P_x = P_x
        if not self.P_x.active:
            return
        if P_x.dim != 4 or int(P_x.shape[1]) != 1 or int(P_x.shape[3]) != 1:
            raise ValueError(f"attention needs whole sequences and heads, [batch, 1, heads, 1], got a partition of shape {list(P_x.shape)}")
        if scale is not None and not scale > 0:
            raise ValueError(f"scale {scale} is not positive")
        _causal_form(causal, own_ends)
        self.causal, self.scale, self.own_ends = bool(causal), scale, bool(own_ends)

    def extra_repr(self) -> str:
        return f'causal={self.causal}, scale={self.scale}, own_ends={self.own_ends}' if self.P_x.active else ''

    def forward(self, q, k, v, lengths=None):
        if not self.P_x.active:
            return q
        return attention_shard(q, k, v, lengths, causal=self.causal, scale=self.scale, own_ends=self.own_ends)
