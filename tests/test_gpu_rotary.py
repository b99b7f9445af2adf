"""Rotation of queries and keys, alone and behind the norm of each head: every layout against the definition in 64 bits.

Tolerances.  Results are rounded once, by at most half a step of their type (``finfo.eps / 2`` of the value; float16 below its
smallest normal number: 2^-25).  Before that, in 32 bits: an angle's rest of a turn is rounded by 2^-26, 2 pi of that is 2^-23.3
of a radian, cosine and sine themselves by 2 units, 2^-23; with the three operations of y = x c - x' s it stays below
2^-21 (|x| + |x'|) amplitude.  A norm's sum of 512 squares, its root and its quotient cost less than 2^-19 of the value, the
adjoint's mean as much again: 2^-18.  Sums over tokens add at most 2^7 terms one after another: 2^-17 of the sum of magnitudes.
"""

import numpy as np
import pytest
import torch

from oracle import heads as o_heads

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
ANGLE, NORM, NORM_ADJOINT, SUM = 2.0 ** -21, 2.0 ** -19, 2.0 ** -18, 2.0 ** -17


def _f64(t):
    return t.detach().double().cpu().numpy()


def _close(got, want, scale, factor):
    """|got - want| <= half a step of the value + factor * scale (and, next to zero, half of float16's smallest step)."""
    dt = got.dtype
    got = _f64(got)
    assert got.shape == want.shape
    step = torch.finfo(dt).eps / 2
    tol = step * np.abs(want) + (1 + step) * factor * scale + (2.0 ** -25 if dt == torch.float16 else 0)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{bad.sum()} of {bad.size} off, worst {np.max(np.abs(got - want) / np.maximum(tol, 1e-300)):.3g} of the tolerance"


def _case(dt, batch, tokens, heads, kv_heads, dim, seed=0, packed=False):
    g = torch.Generator().manual_seed(seed)
    if packed:
        all_ = torch.randn(batch, tokens, (heads + 2 * kv_heads) * dim + 3, generator=g).to(dt).cuda()
        q = all_[..., 1:1 + heads * dim].unflatten(-1, (heads, dim))
        k = all_[..., 1 + heads * dim:1 + (heads + kv_heads) * dim].unflatten(-1, (kv_heads, dim))
    else:
        q = torch.randn(batch, tokens, heads, dim, generator=g).to(dt).cuda()
        k = torch.randn(batch, tokens, kv_heads, dim, generator=g).to(dt).cuda()
    return g, q, k


SHAPES = [   # batch, tokens, heads, kv_heads, dim, rotated
    (1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 8, 8), (1, 5, 3, 1, 64, 64), (2, 33, 8, 1, 128, 128), (1, 7, 5, 5, 80, 32), (3, 2, 2, 1, 100, 100),
    (1, 3, 2, 2, 36, 18), (2, 4, 3, 1, 33, 10), (1, 2, 70, 3, 16, 12), (1, 2, 2, 1, 256, 256), (1, 2, 3, 1, 512, 256), (2, 2, 1, 1, 1, 0),
    (1, 4, 2, 2, 72, 72), (1, 700, 9, 2, 96, 64),
]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("packed", [False, True])
def test_rotation_and_its_adjoint(dt, interleaved, shape, packed):
    from distdl_amd import nn
    batch, tokens, heads, kv_heads, dim, rotated = shape
    g, q, k = _case(dt, batch, tokens, heads, kv_heads, dim, packed=packed)
    freq = nn.rotary_frequencies(rotated, device="cuda")
    positions = torch.randint(0, 1 << 20, (batch, tokens), generator=g).cuda()
    q.requires_grad_(), k.requires_grad_()
    yq, yk = nn.rotary_shard(q, k, freq, positions, interleaved=interleaved, amplitude=1.25)
    dyq, dyk = torch.randn(q.shape, generator=g).to(dt).cuda(), torch.randn(k.shape, generator=g).to(dt).cuda()
    dq, dk = torch.autograd.grad([yq, yk], [q, k], [dyq, dyk])
    f, p = _f64(freq), positions.cpu().numpy()
    for y, x, dx, dy in ((yq, q, dq, dyq), (yk, k, dk, dyk)):
        assert y.is_contiguous()
        _close(y, o_heads.rotate(_f64(x), f, p, interleaved, 1.25), o_heads.pair_sum(_f64(x), len(f), interleaved, 1.25), ANGLE)
        _close(dx, o_heads.rotate(_f64(dy), f, p, interleaved, 1.25, inverse=True), o_heads.pair_sum(_f64(dy), len(f), interleaved, 1.25), ANGLE)
        assert torch.equal(y[..., rotated:], x[..., rotated:])      # what does not turn stays as it is


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("weighted", [False, True])
def test_head_norm_rotation_and_its_adjoint(dt, interleaved, shape, weighted):
    from distdl_amd import nn
    batch, tokens, heads, kv_heads, dim, rotated = shape
    g, q, k = _case(dt, batch, tokens, heads, kv_heads, dim, seed=1, packed=True)
    eps, freq = 1e-5, nn.rotary_frequencies(rotated, device="cuda")
    positions = torch.randint(-50, 1 << 17, (tokens,), generator=g).to(torch.int32).cuda()
    wq, wk = ((1 + 0.3 * torch.randn(dim, generator=g)).to(dt).cuda().requires_grad_() if weighted else None for _ in range(2))
    q.requires_grad_(), k.requires_grad_()
    yq, yk = nn.head_norm_rotary_shard(q, k, wq, wk, freq, positions, eps=eps, interleaved=interleaved)
    dyq, dyk = torch.randn(q.shape, generator=g).to(dt).cuda(), torch.randn(k.shape, generator=g).to(dt).cuda()
    grads = torch.autograd.grad([yq, yk], [q, k] + ([wq, wk] if weighted else []), [dyq, dyk])
    f, p = _f64(freq), positions.cpu().numpy()
    for i, (y, x, w, dy) in enumerate(((yq, q, wq, dyq), (yk, k, wk, dyk))):
        w64 = _f64(w) if weighted else np.ones(dim)
        xhat, rstd = o_heads.head_norm(_f64(x), eps)
        _close(y, o_heads.rotate(xhat * w64, f, p, interleaved), o_heads.pair_sum(xhat * w64, len(f), interleaved), NORM)
        dx, dw = o_heads.head_norm_rotate_backward(_f64(dy), _f64(x), w64, eps, f, p, interleaved)
        g_size = o_heads.pair_sum(_f64(dy), len(f), interleaved)
        wg = g_size * np.abs(w64)
        _close(grads[i], dx, rstd * (wg + np.abs(xhat) * (wg * np.abs(xhat)).mean(-1, keepdims=True)), NORM_ADJOINT)
        if weighted:
            _close(grads[2 + i], dw, (g_size * np.abs(xhat)).sum((0, 1, 2)), SUM)


def test_far_positions_keep_their_angles():
    """A position of 2^40 turns the fastest pair by 64-bit arithmetic: 2^40 radians are exact to 2^-12 of a turn in 53 bits."""
    from distdl_amd import nn
    g, q, _ = _case(torch.float32, 1, 64, 2, 1, 64, seed=3)
    positions = torch.randint(0, 1 << 31, (64,), generator=g).cuda()
    freq = nn.rotary_frequencies(64, device="cuda")
    y, none = nn.rotary_shard(q, None, freq, positions)
    assert none is None
    # 2^31 positions times 2^-53 of the frequency (and of 1 / 2 pi): 2^-21 of a radian more
    _close(y, o_heads.rotate(_f64(q), _f64(freq), positions.cpu().numpy()), o_heads.pair_sum(_f64(q), 32, False), 2 * ANGLE)


def test_positions_none_and_one_row_for_all_sequences():
    from distdl_amd import nn
    _, q, k = _case(torch.bfloat16, 3, 5, 2, 1, 16, seed=4)
    freq = nn.rotary_frequencies(16, device="cuda")
    at = torch.arange(5, device="cuda")
    want = nn.rotary_shard(q, k, freq, at.expand(3, 5))
    for positions in (None, at, at.to(torch.int32), at[None], torch.arange(10, device="cuda")[::2] // 2):
        got = nn.rotary_shard(q, k, freq, positions)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_strided_heads_and_last_dimension():
    """Heads before tokens in memory, a stride in the last dimension, sequences that share their memory."""
    from distdl_amd import nn
    g = torch.Generator().manual_seed(5)
    freq = nn.rotary_frequencies(32, device="cuda")
    base = torch.randn(2, 3, 7, 32, generator=g).cuda()
    for q in (base.transpose(1, 2), torch.randn(2, 7, 3, 64, generator=g).cuda()[..., ::2], base[:1].transpose(1, 2).expand(4, 7, 3, 32)):
        got = nn.rotary_shard(q, None, freq)[0]
        assert torch.equal(got, nn.rotary_shard(q.contiguous(), None, freq)[0])


def test_no_tokens_no_heads_and_unused_outputs():
    from distdl_amd import nn
    freq = nn.rotary_frequencies(8, device="cuda")
    w = torch.ones(8, device="cuda", requires_grad=True)
    for shape in ((0, 3, 2, 8), (2, 0, 2, 8), (2, 3, 0, 8)):
        q = torch.zeros(shape, device="cuda", requires_grad=True)
        y, _ = nn.head_norm_rotary_shard(q, None, w, None, freq)
        assert y.shape == q.shape
        dq, dw = torch.autograd.grad(y.sum(), [q, w])
        assert dq.shape == q.shape and torch.equal(dw, torch.zeros_like(dw))
    q, k = torch.randn(1, 4, 2, 8, device="cuda", requires_grad=True), torch.randn(1, 4, 1, 8, device="cuda", requires_grad=True)
    yq, _ = nn.rotary_shard(q, k, freq)
    dq, dk = torch.autograd.grad(yq.sum(), [q, k], allow_unused=True)
    assert dk is None and dq.shape == q.shape
    _, yk = nn.head_norm_rotary_shard(q, k, w, w, freq)
    assert torch.autograd.grad(yk.sum(), [q], allow_unused=True)[0] is None


def test_zero_heads_with_zero_eps_do_not_reach_the_weights_of_others():
    """eps = 0: a head of another lane group that is not there adds nothing to the weights' gradients."""
    from distdl_amd import nn
    q = torch.randn(1, 3, 3, 8, device="cuda", requires_grad=True)
    w = torch.ones(8, device="cuda", requires_grad=True)
    y, _ = nn.head_norm_rotary_shard(q, None, w, None, nn.rotary_frequencies(8, device="cuda"), eps=0.0)
    for grad in torch.autograd.grad(y.square().sum(), [q, w]):
        assert torch.isfinite(grad).all()


@pytest.mark.parametrize("norm", [False, True])
def test_gradients_against_differences(norm):
    """Central differences of the oracle's own value with step h: their error is h^2 times the third derivative, and the sum's
    rounding 2^-50 / h; with h = 2^-14 and values of order one both stay below 2^-20 of the gradient's scale."""
    from distdl_amd import nn
    g, q, _ = _case(torch.float32, 1, 3, 2, 1, 12, seed=6)
    freq, positions, eps = nn.rotary_frequencies(8, device="cuda"), torch.tensor([3, 900, 77], device="cuda"), 1e-5
    w = (1 + 0.2 * torch.randn(12, generator=g)).cuda().requires_grad_()
    t = torch.randn(q.shape, generator=g).cuda()
    q.requires_grad_()
    y = nn.head_norm_rotary_shard(q, None, w, None, freq, positions, eps=eps)[0] if norm else nn.rotary_shard(q, None, freq, positions)[0]
    dq, = torch.autograd.grad(y, [q], [t])

    def value(x):
        x = o_heads.head_norm(x, eps)[0] * _f64(w) if norm else x
        return (o_heads.rotate(x, _f64(freq), positions.cpu().numpy()) * _f64(t)).sum()

    x, h = _f64(q), 2.0 ** -14
    for at in np.ndindex(*x.shape):
        up, down = x.copy(), x.copy()
        up[at] += h
        down[at] -= h
        assert abs((value(up) - value(down)) / (2 * h) - float(dq[at])) <= 2.0 ** -16 * (1 + np.abs(_f64(t)).max())


def test_second_derivatives_are_refused():
    from distdl_amd import nn
    q = torch.randn(1, 2, 1, 8, device="cuda", requires_grad=True)
    y, _ = nn.rotary_shard(q, None, nn.rotary_frequencies(8, device="cuda"))
    dq, = torch.autograd.grad(y.square().sum(), [q], create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dq.sum(), [q])


def test_equal_calls_give_equal_bits():
    from distdl_amd import nn
    _, q, k = _case(torch.bfloat16, 2, 999, 12, 3, 96, seed=8)
    freq = nn.rotary_frequencies(96, device="cuda")
    w = torch.ones(96, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    q.requires_grad_(), k.requires_grad_()
    runs = []
    for _ in range(2):
        y = nn.head_norm_rotary_shard(q, k, w, w, freq)
        runs.append(torch.autograd.grad(y, [q, k, w], [q.detach(), k.detach()]))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_graph_replays_on_another_stream():
    """Captured on a side stream, replayed with eager work between; forward and adjoint."""
    from distdl_amd import nn
    g, q, k = _case(torch.bfloat16, 2, 40, 4, 2, 64, seed=9)
    freq, positions = nn.rotary_frequencies(64, device="cuda"), torch.arange(40, device="cuda")
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    q.requires_grad_()

    def step():
        yq, yk = nn.head_norm_rotary_shard(q, k, w, w, freq, positions)
        return [yq.detach(), yk.detach()] + list(torch.autograd.grad([yq, yk], [q, w], [yq.detach(), yk.detach()]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    for i in range(3):
        with torch.no_grad():
            q.copy_(torch.randn(q.shape, generator=g).to(q.dtype))
            positions.add_(100 * i)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, want))


def test_layers_broadcast_their_weights_and_take_views():
    from distdl_amd.backends.stub_hip import SimWorld
    from distdl_amd import nn
    P = SimWorld(1).partition(0).create_partition_inclusive([0]).create_cartesian_topology_partition([1, 1, 1, 1])
    layer = nn.DistributedHeadNormRotary(P, 32, rotated=16, scaling="linear", factor=4.0, interleaved=True, dtype=torch.bfloat16)
    _, q, k = _case(torch.bfloat16, 2, 6, 4, 1, 32, seed=10, packed=True)
    with torch.no_grad():
        layer.q_weight.mul_(2)
    yq, yk = layer(q, k)
    freq = nn.rotary_frequencies(16, scaling="linear", factor=4.0, device="cuda")
    want = nn.head_norm_rotary_shard(q, k, 2 * torch.ones(32, dtype=torch.bfloat16, device="cuda"), None, freq, interleaved=True)
    assert torch.equal(yq, want[0]) and torch.equal(yk, want[1])
    (yq.float().sum() + yk.float().sum()).backward()
    assert layer.q_weight.grad.shape == layer.q_weight.shape and layer.k_weight.grad is not None
    plain = nn.DistributedRotary(P, 32, amplitude=1.5).to(torch.float16)       # moves between types leave the angles' 64 bits
    assert torch.equal(plain(q)[0], nn.rotary_shard(q, None, nn.rotary_frequencies(32, device="cuda"), amplitude=1.5)[0])


@pytest.mark.parametrize("norm", [False, True])
def test_keys_alone(norm):
    from distdl_amd import nn
    _, q, k = _case(torch.float16, 2, 9, 2, 3, 24, seed=11)
    freq = nn.rotary_frequencies(24, device="cuda")
    w = torch.full((24,), 1.5, dtype=torch.float16, device="cuda").requires_grad_()

    def call(a, b):
        return nn.head_norm_rotary_shard(a, b, w if a is not None else None, w, freq) if norm else nn.rotary_shard(a, b, freq)

    k.requires_grad_()
    none, alone = call(None, k)
    _, both = call(q, k)
    assert none is None and torch.equal(alone, both)
    for leaf in [k] + ([w] if norm else []):
        assert torch.equal(torch.autograd.grad(alone, [leaf], k.detach(), retain_graph=True)[0], torch.autograd.grad(both, [leaf], k.detach(), retain_graph=True)[0])
    with pytest.raises(ValueError, match="neither"):
        nn.rotary_shard(None, None, freq)
