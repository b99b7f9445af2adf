"""The causal form next to caches of sequences of different lengths: the queries are every sequence's last tokens.  Each sequence against the definition in 64
bits of it alone, cut to its length, with the bounds of the general test."""

import pytest
import torch

from oracle import heads as o_heads
from test_gpu_attention import TYPES
from test_gpu_attention import _bounds
from test_gpu_attention import _f64
from test_gpu_attention import _inputs
from test_gpu_attention import _within

pytestmark = pytest.mark.gpu

CASES = [   # tokens, keys, heads, kv_heads, dim, lengths
    (2, 700, 8, 2, 128, [700, 513, 2, 1, 0]), (4, 1100, 8, 1, 80, [1100, 33, 4, 3, -7, 5000]), (1, 40, 4, 4, 40, [40, 1, 0]), (70, 300, 4, 2, 64, [300, 70, 69, 71, 100, 1]),
    (33, 40, 2, 1, 32, [40, 33, 7]), (200, 200, 2, 2, 96, [200, 31, 130]), (5, 9000, 4, 1, 128, [9000, 4097, 4096]), (130, 520, 16, 2, 72, 5 * [520, 131, 300]), (9, 60, 4, 1, 24, [60, 9, 33]),
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("case", CASES)
def test_queries_are_the_last_tokens_of_their_own_sequence(dt, case):
    from distdl_amd import nn
    tokens, keys, heads, kv_heads, dim, lengths = case
    q, k, v, dy = _inputs(dt, len(lengths), tokens, keys, heads, kv_heads, dim, seed=21)
    for b, n in enumerate(lengths):
        k[b, max(0, n):] = v[b, max(0, n):] = float("nan")      # (not read)
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        alone = nn.attention_shard(q, k, v, n, causal=True, own_ends=True)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = nn.attention_shard(*leaves, n, causal=True, own_ends=True)
    assert torch.equal(out, alone)
    grads = torch.autograd.grad(out, leaves, dy)
    u, tiny = torch.finfo(dt).eps / 2, 2.0 ** -25 if dt == torch.float16 else 0.0
    for b, have in enumerate(lengths):
        have = min(max(have, 0), keys)
        for name, grad in (("dk", grads[1]), ("dv", grads[2])):
            assert not grad[b, have:].any(), name
        if have == 0:
            assert not out[b].any() and not grads[0][b].any()
            continue
        qn, kn, vn, dyn = _f64(q[b:b + 1]), _f64(k[b:b + 1, :have]), _f64(v[b:b + 1, :have]), _f64(dy[b:b + 1])
        want = o_heads.attention(qn, kn, vn, None, True, None, dyn)
        tol = _bounds(qn, kn, vn, None, True, dim ** -0.5, u, tiny, dyn, dt != torch.float32)
        got = (out[b:b + 1], grads[0][b:b + 1], grads[1][b:b + 1, :have], grads[2][b:b + 1, :have])
        for name, g, w, t, more in zip(("out", "dq", "dk", "dv"), got, (want[0],) + want[2:], tol, (0, u, u, u)):
            _within(name, g, w, t, more)


def test_equal_lengths_and_one_token_are_as_before():
    from distdl_amd import nn
    q, k, v, _ = _inputs(torch.bfloat16, 3, 4, 90, 4, 2, 64, seed=22)
    whole = torch.full((3,), 90, dtype=torch.int32, device="cuda")
    want = nn.attention_shard(q, k, v, causal=True)
    for lengths in (None, whole):
        assert torch.equal(nn.attention_shard(q, k, v, lengths, causal=True, own_ends=True), want)
    some = torch.tensor([90, 17, 1], dtype=torch.int32, device="cuda")
    one = nn.attention_shard(q[:, :1], k, v, some)
    assert torch.equal(nn.attention_shard(q[:, :1], k, v, some, causal=True, own_ends=True), one)


def test_the_layer_and_the_general_path():
    from distdl_amd import nn
    from distdl_amd import hip_ops
    from distdl_amd.backends.stub_hip import SimWorld
    from distdl_amd.nn import attention
    P = SimWorld(1).partition(0).create_partition_inclusive([0]).create_cartesian_topology_partition([1, 1, 1, 1])
    q, k, v, dy = _inputs(torch.float16, 2, 3, 50, 4, 1, 36, seed=23)
    lengths = torch.tensor([50, 20], dtype=torch.int32, device="cuda")
    results = []
    for call in (lambda *t: nn.DistributedAttention(P, causal=True, own_ends=True)(*t, lengths), lambda *t: nn.attention_shard(*t, lengths, causal=True, own_ends=True),
                 lambda *t: attention._AttentionShard.apply(*t, lengths, hip_ops.CAUSAL_OWN_ENDS, None)):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = call(*leaves)
        results.append([out.detach()] + list(torch.autograd.grad(out, leaves, dy)))
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
