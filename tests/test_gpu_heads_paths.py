"""The heads' operators through the ways that a program may come in by: the native nodes and the general path behind them (the same bits), gradients
that are views of one element, tensors kept elsewhere, operands changed in between, several threads, an observer of all calls."""

import threading

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu


def _attention(dt, dim, tokens=37, keys=70, seed=0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, dy = (torch.randn(2, n, h, dim, generator=g).to(dt).cuda() for n, h in ((tokens, 4), (keys, 2), (keys, 2), (tokens, 4)))
    return (q, k, v, torch.tensor([keys, 5], dtype=torch.int32, device="cuda")), (dy,)


def _rotary(dt, dim, norm, seed=0):
    from distdl_amd import nn
    g = torch.Generator().manual_seed(seed)
    packed = torch.randn(2, 33, 6 * dim, generator=g).to(dt).cuda()
    q, k = packed[..., :4 * dim].unflatten(-1, (4, dim)), packed[..., 4 * dim:].unflatten(-1, (2, dim))
    weights = [torch.randn(dim, generator=g).to(dt).cuda() for _ in range(2)] if norm else []
    dys = tuple(torch.randn(2, 33, h, dim, generator=g).to(dt).cuda() for h in (4, 2))
    return (q, k, *weights, nn.rotary_frequencies(dim // 4 * 2, device="cuda"), torch.arange(33, device="cuda") + 1000), dys


def _operator(name, dt, dim, seed=0):
    """``(native, general, operands, gradients of the results, how many of the operands are leaves)``."""
    from distdl_amd import nn
    from distdl_amd.nn import attention, rotary
    if name == "attention":
        operands, dys = _attention(dt, dim, seed=seed)
        return (lambda *t: nn.attention_shard(*t, causal=True), lambda *t: attention._AttentionShard.apply(*t, True, None), operands, dys, 3)
    operands, dys = _rotary(dt, dim, name == "head_norm", seed)
    if name == "rotary":
        return (lambda *t: nn.rotary_shard(*t, interleaved=True, amplitude=1.5), lambda *t: rotary._RotaryShard.apply(*t, True, 1.5), operands, dys, 2)
    return (lambda *t: nn.head_norm_rotary_shard(*t, eps=1e-3), lambda *t: rotary._HeadNormRotaryShard.apply(*t, 1e-3, False, 1.0), operands, dys, 4)


def _step(call, operands, dys, count):
    leaves = [t.detach().requires_grad_() for t in operands[:count]]
    out = call(*leaves, *operands[count:])
    out = out if isinstance(out, tuple) else (out,)
    return [o.detach() for o in out] + list(torch.autograd.grad(out, leaves, dys))


def _same(a, b):
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


OPERATORS = ["attention", "rotary", "head_norm"]


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [33, 64, 100])
@pytest.mark.parametrize("name", OPERATORS)
def test_native_and_general_paths_give_the_same_bits(name, dim, dt):
    native, general, operands, dys, count = _operator(name, dt, dim)
    want = _step(native, operands, dys, count)
    assert _same(want, _step(general, operands, dys, count))
    detached = native(*operands)
    assert _same(want[:len(dys)], detached if isinstance(detached, tuple) else (detached,))


@pytest.mark.parametrize("name", OPERATORS)
def test_gradients_of_a_sum_are_views_of_one_element(name):
    native, _, operands, dys, count = _operator(name, torch.bfloat16, 64)
    ones = [torch.ones_like(dy) for dy in dys]
    assert _same(_step(native, operands, ones, count), _step(native, operands, [torch.ones((), dtype=dy.dtype, device="cuda").expand(dy.shape) for dy in dys], count))


@pytest.mark.parametrize("dim", [64, 100])
@pytest.mark.parametrize("name", OPERATORS)
def test_kept_tensors_may_leave_the_card(name, dim):
    native, _, operands, dys, count = _operator(name, torch.float16, dim)
    want = _step(native, operands, dys, count)
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
        assert _same(want, _step(native, operands, dys, count))


@pytest.mark.parametrize("name", ["attention", "head_norm"])
def test_operands_that_change_before_the_adjoint_are_an_error(name):
    native, _, operands, dys, count = _operator(name, torch.bfloat16, 64)
    operands = [t.detach().clone() for t in operands]
    leaves = [t.requires_grad_() for t in operands[:count]]
    out = native(*leaves, *operands[count:])
    with torch.no_grad():
        leaves[0].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaves, dys)


def test_a_result_that_changes_before_the_adjoint_is_an_error():
    native, _, operands, dys, count = _operator("attention", torch.bfloat16, 64)
    leaves = [t.detach().requires_grad_() for t in operands[:count]]
    out = native(*leaves, *operands[count:])
    with torch.no_grad():
        out.mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaves, dys)


def test_the_same_heads_as_queries_keys_and_values():
    """One leaf three times: its gradient is the sum of the three."""
    from distdl_amd import nn
    x = torch.randn(2, 50, 2, 32, device="cuda")
    dy = torch.randn(2, 50, 2, 32, device="cuda")
    leaf, parts = x.clone().requires_grad_(), [x.clone().requires_grad_() for _ in range(3)]
    got, = torch.autograd.grad(nn.attention_shard(leaf, leaf, leaf, causal=True), [leaf], dy)
    dq, dk, dv = torch.autograd.grad(nn.attention_shard(*parts, causal=True), parts, dy)
    # (three terms in one of their orders: two roundings of half a step of partial sums each)
    assert ((got - (dq + dk + dv)).abs() <= 4 * 2.0 ** -24 * (dq.abs() + dk.abs() + dv.abs())).all()


def test_two_steps_back_through_one_graph_and_only_one_result():
    for name in OPERATORS:
        native, _, operands, dys, count = _operator(name, torch.bfloat16, 64)
        leaves = [t.detach().requires_grad_() for t in operands[:count]]
        out = native(*leaves, *operands[count:])
        out = out if isinstance(out, tuple) else (out,)
        first = torch.autograd.grad(out, leaves, dys, retain_graph=True)
        assert _same(first, torch.autograd.grad(out, leaves, dys, retain_graph=True))
        if len(out) == 2:      # queries alone: no gradient of the keys
            some = torch.autograd.grad(out[0], leaves, dys[0], allow_unused=True)
            assert torch.equal(some[0], first[0]) and (some[1] is None or not some[1].any())
            if count == 4:
                assert torch.equal(some[2], first[2]) and (some[3] is None or not some[3].any())


def test_threads_with_streams_of_their_own():
    """Four threads, each with shapes and a stream of its own, ten steps each: as one after the other."""
    cases = [_operator(name, dt, dim, seed) for seed, (name, dt, dim) in enumerate(
        (("attention", torch.bfloat16, 64), ("attention", torch.float32, 100), ("head_norm", torch.bfloat16, 96), ("rotary", torch.float16, 40)))]
    wants = [_step(c[0], *c[2:]) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(case, want):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(10):
                got = _step(case[0], *case[2:])
                stream.synchronize()
                if not _same(got, want):
                    wrong.append(case)

    threads = [threading.Thread(target=work, args=a) for a in zip(cases, wants)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("name", OPERATORS)
def test_an_observer_of_all_calls(name):
    class Observer(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            return func(*args, **(kwargs or {}))

    native, _, operands, dys, count = _operator(name, torch.bfloat16, 64)
    want = _step(native, operands, dys, count)
    with Observer():
        assert _same(want, _step(native, operands, dys, count))
