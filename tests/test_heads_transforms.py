"""Tangents, traces and transforms that meet the heads' operators where no operand takes a gradient: they see the torch.autograd.Functions, so that nothing
is dropped.  No GPU: the kernels' calls are replaced by definitions in NumPy, which torch does not see either."""

import numpy as np
import pytest
import torch

from distdl_amd import hip_ops
from distdl_amd import nn
from oracle import heads as o_heads


def _numpy(t):
    return t.detach().numpy()


@pytest.fixture
def kept(monkeypatch):
    """The kernels' calls in NumPy; a list of what was asked to be kept for an adjoint."""
    asked = []

    def attention(q, k, v, lengths=None, causal=False, scale=None, want_lse=False):
        asked.append(want_lse)
        out, lse = o_heads.attention(_numpy(q), _numpy(k), _numpy(v), None if lengths is None else _numpy(lengths), causal, scale)
        out = torch.from_numpy(out.astype(np.float32))
        return (out, torch.from_numpy(lse.transpose(0, 2, 1).astype(np.float32).copy()), None) if want_lse else out

    def head_rotary(q, k, frequencies, positions=None, interleaved=False, amplitude=1.0, inverse=False, norm=False, q_weight=None, k_weight=None, eps=1e-6):
        def one(x, w):
            if x is None:
                return None
            at = np.arange(x.shape[1]) if positions is None else _numpy(positions)
            x = o_heads.head_norm(_numpy(x), eps)[0] * (1 if w is None else _numpy(w)) if norm else _numpy(x)
            return torch.from_numpy(o_heads.rotate(x, _numpy(frequencies), at, interleaved, amplitude, inverse).astype(np.float32))
        return one(q, q_weight), one(k, k_weight)

    monkeypatch.setattr(hip_ops, "attention", attention)
    monkeypatch.setattr(hip_ops, "head_rotary", head_rotary)
    return asked


def _operator(name):
    """``(call of one tensor, the name of its function)``."""
    freq, w = nn.rotary_frequencies(8), torch.full((8,), 1.5)
    return {"attention": (lambda x: nn.attention_shard(x, x, x, causal=True), "_AttentionShard"),
            "rotary": (lambda x: nn.rotary_shard(x, None, freq)[0], "_RotaryShard"),
            "head_norm": (lambda x: nn.head_norm_rotary_shard(x, None, w, None, freq)[0], "_HeadNormRotaryShard")}[name]


OPERATORS = ["attention", "rotary", "head_norm"]


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("name", OPERATORS)
def test_tangents_are_not_dropped(kept, name, grad_mode):
    call, _ = _operator(name)
    x = torch.randn(1, 3, 2, 8)
    with torch.set_grad_enabled(grad_mode), torch.autograd.forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
            call(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", OPERATORS)
def test_traces_hold_the_call(kept, name):
    call, function = _operator(name)
    first, second = torch.randn(1, 3, 2, 8), torch.randn(1, 3, 2, 8)
    traced = torch.jit.trace(call, (first,), check_trace=False)
    assert function in str(traced.graph)
    assert torch.equal(traced(second), call(second))


@pytest.mark.parametrize("name", OPERATORS)
def test_calls_without_gradients_keep_nothing(kept, name):
    call, _ = _operator(name)
    x, leaf = torch.randn(1, 3, 2, 8), torch.randn(1, 3, 2, 8, requires_grad=True)
    assert not call(x).requires_grad and call(leaf).requires_grad
    with torch.no_grad():
        assert not call(leaf).requires_grad
    assert kept == ([False, True, False] if name == "attention" else [])


def test_neither_queries_nor_keys_is_refused():
    freq = nn.rotary_frequencies(8)
    for call in (lambda: nn.rotary_shard(None, None, freq), lambda: nn.head_norm_rotary_shard(None, None, None, None, freq)):
        with pytest.raises(ValueError, match="neither"):
            call()


def test_own_ends_belong_to_the_causal_form():
    from distdl_amd.backends.stub_hip import SimWorld
    q = torch.zeros(1, 2, 2, 8)
    P = SimWorld(1).partition(0).create_partition_inclusive([0]).create_cartesian_topology_partition([1, 1, 1, 1])
    for call in (lambda: nn.attention_shard(q, q, q, own_ends=True), lambda: nn.DistributedAttention(P, own_ends=True)):
        with pytest.raises(ValueError, match="own_ends"):
            call()
    assert "own_ends=True" in repr(nn.DistributedAttention(P, causal=True, own_ends=True))
