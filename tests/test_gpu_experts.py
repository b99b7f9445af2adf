"""Tokens to their experts and back against the 64-bit oracle."""

import numpy as np
import pytest
import torch

from distdl_amd import hip_ops
from distdl_amd import nn
from oracle import experts as o

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def n64(t):
    return t.detach().double().cpu().numpy()


def choices(rng, tokens, chosen, experts, kind="any"):
    ids = rng.integers(0, max(1, experts), (tokens, chosen))
    if kind == "one":
        ids[:] = experts // 2
    if kind == "padded":
        ids[tokens // 2:] = -1
    if kind == "wild":
        ids = rng.choice([-2 ** 40, -1, 0, 1, experts - 1, experts, 2 ** 33, 2 ** 32 + 1], (tokens, chosen))
    return ids


@pytest.mark.parametrize("tokens,chosen,experts,window,kind", [
    (0, 2, 4, None, "any"), (1, 1, 1, None, "any"), (5, 0, 3, None, "any"), (3, 2, 0, None, "any"), (7, 3, 5, (2, 2), "any"), (16, 2, 8, None, "any"),
    (64, 1, 64, None, "any"), (65, 4, 63, (1, 62), "any"), (511, 3, 13, (2, 11), "padded"), (1000, 4, 7, None, "one"), (4096, 1, 300, None, "any"),
    (1024, 4, 128, None, "any"), (4097, 1, 5, None, "any"), (2049, 3, 2047, None, "any"), (3000, 8, 256, (32, 64), "any"), (20001, 3, 40, None, "padded"),
    (9000, 2, 6, None, "one"), (700, 5, 12, (0, 12), "wild"), (5000, 2, 12, (3, 12), "wild"), (40000, 8, 2047, None, "any")])
@pytest.mark.parametrize("index", [torch.int32, torch.int64], ids=["int32", "int64"])
def test_plan(tokens, chosen, experts, window, kind, index):
    ids = choices(np.random.default_rng(tokens * 7 + chosen), tokens, chosen, experts, kind)
    if index == torch.int32:
        ids = ids.astype(np.int32)
    plan = nn.expert_plan(torch.from_numpy(ids).cuda(), experts, window=window)
    low, high = window or (0, experts)
    place, offsets = o.plan(ids, low, high)
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
    assert np.array_equal(plan.place.cpu().numpy(), place)


def test_plan_of_strided_choices():
    ids = torch.randint(0, 9, (300, 6), device="cuda")
    for view in (ids[:, 1:4], ids[::3], ids.t()[:4], ids[:, ::2]):
        place, offsets = o.plan(view.cpu().numpy(), 0, 9)
        plan = nn.expert_plan(view, 9)
        assert np.array_equal(plan.place.cpu().numpy(), place) and np.array_equal(plan.offsets.cpu().numpy(), offsets)


MOVES = [(1, 1, 1, 1), (3, 2, 4, 5), (16, 2, 8, 64), (7, 3, 5, 100), (33, 4, 6, 1001), (65, 1, 3, 8), (5, 8, 16, 2048), (130, 2, 4, 257), (9, 2, 3, 8192), (40, 3, 7, 16), (2, 2, 2, 9000)]


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("tokens,chosen,experts,cols", MOVES)
def test_there_and_back_with_gradients(tokens, chosen, experts, cols, dtype):
    rng = np.random.default_rng(tokens + cols)
    ids = choices(rng, tokens, chosen, experts)
    ids[tokens // 3] = -1
    window = (1, experts) if experts > 2 else (0, experts)
    g = torch.Generator().manual_seed(cols)
    x, y, dm, dout = ((torch.randn(n, cols, generator=g)).to(dtype).cuda() for n in (tokens, tokens * chosen, tokens * chosen, tokens))
    weights = torch.rand(tokens, chosen, generator=g).cuda()
    plan = nn.expert_plan(torch.from_numpy(ids).cuda(), experts, window=window)
    place, offsets = o.plan(ids, *window)
    held = offsets[-1]
    y[held:] = float("nan")          # nobody's rows are not read
    dm[held:] = float("inf")
    for t in (x, y, weights):
        t.requires_grad_()
    moved, out = nn.expert_sort(x, plan), nn.expert_combine(y, plan, weights)
    assert np.array_equal(n64(moved), o.sort(n64(x), place, held))
    terms = o.combine(np.abs(n64(y)), place, held, n64(weights))
    want = o.combine(n64(y), place, held, n64(weights))
    assert (np.abs(n64(out) - want) <= half(dtype) * np.abs(want) + 2 * chosen * U * terms + 2.0 ** -25).all()
    dx, dy, dw = torch.autograd.grad([moved, out], [x, y, weights], [dm, dout])
    want = o.combine(n64(dm), place, held)
    terms = o.combine(np.abs(n64(dm)), place, held)
    assert (np.abs(n64(dx) - want) <= half(dtype) * np.abs(want) + chosen * U * terms + 2.0 ** -25).all()
    want_dy, want_dw = o.combine_backward(n64(dout), n64(y), place, held, n64(weights))
    assert (np.abs(n64(dy) - want_dy) <= (half(dtype) + U) * np.abs(want_dy) + 2.0 ** -25).all()
    _, terms = o.combine_backward(np.abs(n64(dout)), np.abs(n64(y)), place, held, n64(weights))
    assert (np.abs(n64(dw) - want_dw) <= (cols + 2) * U * terms).all()     # any order of the sum
    again = torch.autograd.grad(nn.expert_combine(y, plan, weights), [y, weights], dout)
    assert torch.equal(again[0], dy) and torch.equal(again[1], dw)


@pytest.mark.parametrize("tokens,chosen,cols", [(1, 1, 1), (5, 2, 16), (9, 3, 31), (33, 8, 2048), (4, 2, 5000)])
def test_rows_in_8_bits_travel_with_their_scales(tokens, chosen, cols):
    rng = np.random.default_rng(cols)
    ids = choices(rng, tokens, chosen, 6)
    plan = nn.expert_plan(torch.from_numpy(ids).cuda(), 6, window=(1, 5))
    codes, scales = nn.quantize_rows(torch.randn(tokens, cols, generator=torch.Generator().manual_seed(1)).cuda())
    rows, row_scales = nn.expert_sort(codes, plan, scales)
    place, offsets = o.plan(ids, 1, 5)
    assert rows.dtype == torch.float8_e4m3fn
    assert np.array_equal(rows.view(torch.uint8).cpu().numpy(), o.sort(codes.view(torch.uint8).cpu().numpy(), place, offsets[-1]))
    assert np.array_equal(row_scales.cpu().numpy(), o.sort(scales.cpu().numpy()[:, None], place, offsets[-1])[:, 0])


def test_strided_rows_and_gradients_of_one_side():
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 4, (10, 2), generator=g).cuda()
    plan = nn.expert_plan(ids, 4)
    place, offsets = o.plan(ids.cpu().numpy(), 0, 4)
    x = torch.randn(10, 50, generator=g).cuda()[:, 7:40]
    assert np.array_equal(n64(nn.expert_sort(x, plan)), o.sort(n64(x), place, 20))
    y = torch.randn(33, 20, generator=g).cuda().t()
    np.testing.assert_allclose(n64(nn.expert_combine(y, plan)), o.combine(n64(y), place, 20), rtol=1e-6, atol=1e-6)
    dout, weights = torch.randn(10, 33, generator=g).cuda(), torch.rand(10, 2, generator=g).cuda()
    want = o.combine_backward(n64(dout), n64(y), place, 20, n64(weights))
    for need_y, need_w in ((True, False), (False, True)):
        a, b = y.clone().requires_grad_(need_y), weights.clone().requires_grad_(need_w)
        (grad,) = torch.autograd.grad(nn.expert_combine(a, plan, b), [a if need_y else b], dout)
        np.testing.assert_allclose(n64(grad), want[0 if need_y else 1], rtol=1e-5, atol=1e-5)
    a = y.clone().requires_grad_()
    (grad,) = torch.autograd.grad(nn.expert_combine(a, plan), [a], dout)
    assert np.array_equal(n64(grad), o.sort(n64(dout), place, 20))


def test_captured_and_replayed():
    g = torch.Generator().manual_seed(4)
    ids = torch.randint(0, 16, (3000, 2), generator=g).cuda()
    x, weights = torch.randn(3000, 64, generator=g).cuda(), torch.rand(3000, 2, generator=g).cuda()

    def step():
        place, offsets = hip_ops.expert_plan(ids, 2, 14)
        moved = hip_ops.expert_sort(x, place, offsets)[0]
        return (place, offsets, moved, hip_ops.expert_combine(moved, place, offsets, weights)) + hip_ops.expert_combine_backward(x, moved, place, offsets, weights)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        ids.copy_(torch.randint(0, 16, (3000, 2), generator=torch.Generator().manual_seed(seed)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step()))


@pytest.mark.parametrize("tokens,chosen,experts,window,cols", [(1, 1, 1, None, 3), (37, 3, 5, (1, 4), 65), (300, 2, 8, None, 128)])
def test_gradients_against_differences(tokens, chosen, experts, window, cols):
    """The way there, a product and the way back are linear in every operand, so a difference of any width is the gradient times the step."""
    g = torch.Generator().manual_seed(tokens)
    plan = nn.expert_plan(torch.randint(0, experts, (tokens, chosen), generator=g).cuda(), experts, window=window)
    held = len(plan.offsets) - 1
    operands = [torch.randn(*s, generator=g).cuda() for s in ((tokens, cols), (held, 24, cols), (tokens, chosen))]
    dout = torch.randn(tokens, 24, generator=g).cuda()

    def run(x, w, weights):
        return nn.expert_combine(nn.expert_linear_shard(nn.expert_sort(x, plan), w, plan.offsets), plan, weights)

    leaves = [t.clone().requires_grad_() for t in operands]
    grads = torch.autograd.grad(run(*leaves), leaves, dout)
    for i, grad in enumerate(grads):
        step = torch.randn(operands[i].shape, generator=g).cuda()
        far = [t + step if j == i else t for j, t in enumerate(operands)]
        moved = far[i].double() - operands[i].double()       # the step as the sum was rounded
        change = ((run(*far).double() - run(*operands).double()) * dout.double()).sum()
        # results: sums of cols and chosen terms, the weight and the rows rounded on the way; of the terms' sizes, at both ends; gradients as much again
        sizes = (run(*[t.abs() for t in operands]).double() + run(*[t.abs() for t in far]).double())
        bound = 4 * (cols + chosen + tokens * chosen + 8) * U * (sizes * dout.abs()).sum()
        assert (change - (grad.double() * moved).sum()).abs() <= bound
