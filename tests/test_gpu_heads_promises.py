"""What the heads' operators promise beside their values: results in the place of operands, workers that share the tokens, positions far away, and passes that
torch records before it runs them."""

import numpy as np
import pytest
import torch

from oracle import heads as o_heads

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _heads(dt, batch=3, tokens=70, heads=5, kv_heads=2, dim=96, seed=0):
    """Views of one tensor, with something between and behind them."""
    g = torch.Generator().manual_seed(seed)
    packed = torch.randn(batch, tokens, (heads + kv_heads) * dim + 11, generator=g).to(dt).cuda()
    return packed, packed[..., 3:3 + heads * dim].unflatten(-1, (heads, dim)), packed[..., 5 + heads * dim:5 + (heads + kv_heads) * dim].unflatten(-1, (kv_heads, dim))


def _strides(t):
    from distdl_amd import _lib
    return _lib.i64_array(t.stride()[:3])


def _codes(dt):
    from distdl_amd import _lib
    return {torch.float32: _lib.DDL_DT_F32, torch.bfloat16: _lib.DDL_DT_BF16, torch.float16: _lib.DDL_DT_F16}[dt]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("norm", [0, 1])
@pytest.mark.parametrize("neighbours", [0, 1])
@pytest.mark.parametrize("dim,rotated", [(96, 64), (33, 10), (128, 128), (36, 18)])
@pytest.mark.parametrize("tokens,heads", [(1, 70), (70, 5), (1500, 2)])
def test_rotation_in_the_place_of_its_operands(dt, norm, neighbours, dim, rotated, tokens, heads):
    """The bits of a call with results of their own, and nothing beside the heads is touched."""
    from distdl_amd import _lib
    from distdl_amd import hip_ops
    from distdl_amd import nn
    freq = nn.rotary_frequencies(rotated, device="cuda")
    packed, q, k = _heads(dt, tokens=tokens, heads=heads, dim=dim)
    batch, w = q.shape[0], torch.linspace(0.5, 2, dim).to(dt).cuda() if norm else None
    want = hip_ops.head_rotary(q, k, freq, None, bool(neighbours), 1.0, norm=bool(norm), q_weight=w, k_weight=w, eps=1e-6)
    rest = packed.clone()
    _lib.check(_lib.load().ddl_head_rotary(
        q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), _codes(dt), batch, tokens, heads, k.shape[2], dim, hip_ops._ptr(w), hip_ops._ptr(w), norm, 1e-6,
        freq.data_ptr(), rotated, None, 0, 0, neighbours, 1.0, 0, q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), hip_ops._stream()), "ddl_head_rotary")
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
    for t in (packed, rest):
        t[..., 3:3 + heads * dim], t[..., 5 + heads * dim:5 + (heads + k.shape[2]) * dim] = 0, 0
    assert torch.equal(packed, rest)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("place", ["gradients", "heads"])
@pytest.mark.parametrize("dim,rotated,tokens,heads", [(96, 64, 70, 5), (33, 10, 1, 70), (128, 128, 1500, 2)])
def test_adjoint_of_head_norms_in_the_place_of_its_operands(dt, place, dim, rotated, tokens, heads):
    from distdl_amd import _lib
    from distdl_amd import hip_ops
    from distdl_amd import nn
    freq = nn.rotary_frequencies(rotated, device="cuda")
    (_, q, k), (_, dyq, dyk) = _heads(dt, tokens=tokens, heads=heads, dim=dim), _heads(dt, tokens=tokens, heads=heads, dim=dim, seed=1)
    w = torch.linspace(0.5, 2, dim).to(dt).cuda()
    want = hip_ops.head_norm_rotary_backward(dyq, dyk, q, k, w, w, freq, want_q_weight=True, want_k_weight=True)
    lib = _lib.load()
    elems = lib.ddl_head_norm_rotary_backward_workspace(dim)
    work, dqw, dkw = torch.full((elems,), float("nan"), device="cuda"), torch.empty_like(w), torch.empty_like(w)
    dq, dk = (dyq, dyk) if place == "gradients" else (q, k)
    _lib.check(lib.ddl_head_norm_rotary_backward(
        dyq.data_ptr(), _strides(dyq), dyk.data_ptr(), _strides(dyk), q.data_ptr(), _strides(q), k.data_ptr(), _strides(k), _codes(dt), q.shape[0], tokens, heads,
        k.shape[2], dim, w.data_ptr(), w.data_ptr(), 1e-6, freq.data_ptr(), rotated, None, 0, 0, 0, 1.0, dq.data_ptr(), _strides(dq), dk.data_ptr(), _strides(dk),
        dqw.data_ptr(), dkw.data_ptr(), work.data_ptr(), elems, hip_ops._stream()), "ddl_head_norm_rotary_backward")
    assert all(torch.equal(a, b) for a, b in zip((dq, dk, dqw, dkw), want))


def test_workers_that_share_the_tokens():
    """Two of them, each with the positions of its own tokens: the whole's bits, and weights' gradients that are sums of another order (2^-17 of the
    magnitudes, as for one worker's own)."""
    from distdl_amd import nn
    from distdl_amd.backends.stub_hip import SimWorld
    g = torch.Generator().manual_seed(2)
    q, k, dyq, dyk = (torch.randn(2, 46, h, 32, generator=g) for h in (4, 2, 4, 2))

    def body(P_world, workers):
        P = P_world.create_partition_inclusive(list(range(workers))).create_cartesian_topology_partition([1, workers, 1, 1])
        if not P.active:
            return None
        norm, plain = nn.DistributedHeadNormRotary(P, 32, rotated=16, interleaved=True), nn.DistributedRotary(P, 32, amplitude=1.5)

        def own(t, dim=1):
            return t.chunk(workers, dim)[int(P.index[1])].contiguous().cuda()
        at = own(torch.arange(46) + 1000, 0)
        a, b = own(q).requires_grad_(), own(k).requires_grad_()
        y = norm(a, b, positions=at)
        torch.autograd.backward(y, [own(dyq), own(dyk)])
        z = plain(a.detach(), b.detach(), positions=at)
        return int(P.index[1]), [t.detach().cpu() for t in (*y, a.grad, b.grad, *z)], [None if w.grad is None else w.grad.cpu() for w in (norm.q_weight, norm.k_weight)]

    whole = SimWorld(1).run(lambda P: body(P, 1))[0]
    parts = SimWorld(2).run(lambda P: body(P, 2))
    for index, mine, _ in parts:
        for a, b in zip(mine, whole[1]):
            assert torch.equal(a, b.chunk(2, 1)[index])
    for got, want, heads in zip(parts[0][2], whole[2], (4, 2)):
        assert (got - want).abs().max() <= 2.0 ** -17 * 2 * 46 * heads * want.abs().max()


@pytest.mark.parametrize("power", [33, 40, 46])
def test_positions_of_many_digits(power):
    """Positions up to 2^power.  An angle in turns is a product of two rounded factors and rounded itself, 3 2^-53 of up to 2^power / 2 pi turns: 3 2^(power - 53) radians
    for the fastest pair; the oracle's own product 2^(power - 53)."""
    from distdl_amd import nn
    g = torch.Generator().manual_seed(power)
    q = torch.randn(2, 64, 2, 64, generator=g).cuda()
    positions = torch.randint(1 << (power - 1), 1 << power, (2, 64), generator=g)
    freq = nn.rotary_frequencies(64)
    got = nn.rotary_shard(q, None, freq.cuda(), positions.cuda())[0].double().cpu().numpy()
    x = q.double().cpu().numpy()
    want = o_heads.rotate(x, freq.numpy(), positions.numpy())
    bound = 2.0 ** -24 * np.abs(want) + (2.0 ** -21 + 4 * 2.0 ** (power - 53)) * o_heads.pair_sum(x, 32, False)
    assert (np.abs(got - want) <= bound).all()


def _operators():
    """Name: (call of the leaves, leaves, gradients of the results)."""
    from distdl_amd import nn
    g = torch.Generator().manual_seed(3)
    q, k, v, dy = (torch.randn(2, n, h, 40, generator=g).to(torch.bfloat16).cuda() for n, h in ((21, 4), (50, 2), (50, 2), (21, 4)))
    rq, rk, dyq, dyk = (torch.randn(2, 21, h, 40, generator=g).to(torch.bfloat16).cuda() for h in (4, 2, 4, 2))
    w = torch.linspace(0.5, 2, 40).to(torch.bfloat16).cuda()
    lengths, at, freq = torch.tensor([50, 7], dtype=torch.int32, device="cuda"), torch.arange(21, device="cuda") + 5, nn.rotary_frequencies(20, device="cuda")
    return {
        "attention": (lambda *t: nn.attention_shard(*t), [q, k, v], [dy]),
        "attention_lengths": (lambda *t: nn.attention_shard(*t, lengths, causal=True, own_ends=True), [q, k, v], [dy]),
        "attention_padded": (lambda *t: nn.attention_shard(*t, lengths), [t[..., :33] for t in (q, k, v)], [dy[..., :33]]),
        "rotary": (lambda *t: nn.rotary_shard(*t, freq), [rq, rk], [dyq, dyk]),
        "rotary_positions": (lambda *t: nn.rotary_shard(*t, freq, at, interleaved=True, amplitude=1.5), [rq, rk], [dyq, dyk]),
        "rotary_queries": (lambda t: nn.rotary_shard(t, None, freq)[0], [rq], [dyq]),
        "head_norm": (lambda *t: nn.head_norm_rotary_shard(*t, freq, at), [rq, rk, w, w * 2], [dyq, dyk]),
        "head_norm_plain": (lambda *t: nn.head_norm_rotary_shard(*t, None, None, freq), [rq, rk], [dyq, dyk]),
        "head_norm_keys": (lambda t, u: nn.head_norm_rotary_shard(None, t, None, u, freq)[1], [rk, w], [dyk]),
    }


def _passes(name, seed):
    """All results with their gradients; each result alone; one leaf at a time."""
    call, operands, dys = _operators()[name]
    leaves = [t.detach().clone().requires_grad_() for t in operands]
    out = call(*leaves)
    out = list(out) if isinstance(out, tuple) else [out]
    dys = [seed * dy for dy in dys]
    passes = [[o.detach() for o in out], torch.autograd.grad(out, leaves, dys, retain_graph=True)]
    passes += [torch.autograd.grad([o], leaves, [dy], retain_graph=True, allow_unused=True) for o, dy in zip(out, dys)]
    passes += [torch.autograd.grad(out, [leaf], dys, retain_graph=True) for leaf in leaves]
    for leaf in leaves:
        leaf.grad = None
    torch.autograd.backward(out, dys)
    return passes + [[leaf.grad for leaf in leaves]]


@pytest.mark.parametrize("name", ["attention", "attention_lengths", "attention_padded", "rotary", "rotary_positions", "rotary_queries", "head_norm", "head_norm_plain", "head_norm_keys"])
def test_compiled_autograd_gives_the_bits_of_an_ordinary_pass(name):
    """As it is recorded and with other values, also where one of two results is not used (its gradient never comes) and where there are no positions, lengths,
    weights, queries or keys."""
    from torch._dynamo import compiled_autograd
    want = [_passes(name, seed) for seed in (1, 2)]
    with compiled_autograd._enable(lambda graph: graph):
        got = [_passes(name, seed) for seed in (1, 2)]
    for a, b in zip(got, want):
        assert len(a) == len(b)
        for x, y in zip(a, b):
            for s, t in zip(x, y):
                assert (s is None or not s.any()) if t is None else (torch.equal(s, t) if s is not None else not t.any())
