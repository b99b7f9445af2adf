"""The experts' products and their adjoint against the 64-bit oracle, and a block of all of these operators."""

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


def near(got, want, terms, depth, dtype, in_eights=0.0):
    """A sum of ``depth`` products in 32 bits, in any order, and the result's rounding (the smallest steps of fp16 aside)."""
    off = np.abs(n64(got) - want)
    assert (off <= half(dtype) * np.abs(want) + (2 * (depth + 2) * U + in_eights) * terms + 2.0 ** -25).all(), (off - half(dtype) * np.abs(want)).max()


# The matrix cores add e4m3 products in eights, whose members they cut off at 2^-13 of the largest one's power of two (one product of 2^16 next to one of 2^e
# gives their sum down to e = 3 inside an eight, as float32 does to e = -7 between two of them): up to seven members are off by less than 2^-13 of the largest,
# which is at most the sum of all eight sizes, so a result is off by less than 7 2^-13 of the sum of its terms' sizes.
IN_EIGHTS = 7 * 2.0 ** -13


# counts, spare rows, in, out
CASES = [
    ([1], 0, 8, 8), ([0], 3, 16, 24), ([0, 0, 5], 0, 64, 40), ([3, 0, 2, 1], 4, 128, 96), ([16, 1, 0, 33, 7], 0, 264, 72), ([40, 9], 2, 1000, 100), ([1, 2, 3], 0, 72, 520),
    ([200, 0, 57, 130], 11, 320, 264), ([300, 513], 0, 136, 264), ([700, 0, 900], 5, 512, 768), ([2100, 1500], 0, 256, 512), ([5] * 70, 1, 64, 32),
    # what fills the chip with large tiles: results, gradients of the rows, of the weights
    ([3001, 0, 1200], 7, 72, 8000), ([3001, 0, 1200], 7, 8000, 72), ([9, 0, 130, 2, 64, 1, 70, 200], 3, 2056, 2040),
    # fp32 on the bf16 matrix cores' tiles
    ([513, 0, 600, 490], 3, 1100, 1000), ([400, 0, 700], 0, 2050, 2049),
    # few rows of fp32 by wavefronts on parts of the reduction, up to four blocks of sixteen
    ([30] * 8, 0, 260, 1000), ([8, 1, 0, 20] * 2, 5, 260, 1000), ([1], 0, 8192, 40), ([14, 15], 0, 36, 500),
    # few rows for most: their gradients by wavefronts on parts of the reduction, sixteen at a time
    ([40, 1, 0, 2, 5, 1, 1], 3, 264, 72), ([33, 1, 0, 2, 1, 1, 1], 0, 77, 65), ([2] * 70, 1, 136, 1000), ([16], 0, 4100, 520), ([3] * 64, 0, 600, 40),
    # rows that are no multiple of 16 bytes
    ([5, 0, 9], 2, 9, 11), ([100, 37], 3, 77, 65), ([260, 300], 0, 513, 331), ([1, 1], 0, 1001, 15)]


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("counts,spare,k,n", CASES, ids=[f"{sum(c)}+{s}of{len(c)}-{k}x{n}" for c, s, k, n in CASES])
def test_products_and_adjoint(counts, spare, k, n, dtype):
    g = torch.Generator().manual_seed(k * 3 + n)
    rows, held = sum(counts) + spare, sum(counts)
    x, w, dy = ((torch.randn(*s, generator=g)).to(dtype).cuda() for s in ((rows, k), (len(counts), n, k), (rows, n)))
    x[held:], dy[held:] = float("nan"), float("inf")        # nobody's
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    for t in (x, w):
        t.requires_grad_()
    y = nn.expert_linear_shard(x, w, torch.from_numpy(offsets).cuda())
    dx, dw = torch.autograd.grad(y, [x, w], dy)
    zx, zdy = n64(x), n64(dy)
    zx[held:], zdy[held:] = 0, 0
    want, terms = o.product(zx, n64(w), offsets, zdy), o.product(np.abs(zx), np.abs(n64(w)), offsets, np.abs(zdy))
    near(y, want[0], terms[0], k, dtype)
    near(dx, want[1], terms[1], n, dtype)
    near(dw, want[2], terms[2], max(counts), dtype)
    again = torch.autograd.grad(nn.expert_linear_shard(x, w, torch.from_numpy(offsets).cuda()), [x, w], dy)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


# few rows for most experts, or for all; from 65 (fp32) or 257 rows on the others' own launch, with more experts than a wavefront has lanes; no rows at all; matrices that are no whole
# vectors or lines, and of the smallest sizes
FEW = [([2, 1, 0, 4], 0, 256, 264), ([32, 0, 1], 0, 72, 130), ([33, 0, 1], 3, 72, 130), ([40, 1, 0, 2, 100, 0, 3, 1, 1, 70, 5, 5, 2, 33, 1], 9, 520, 1096), ([0] * 69 + [20], 0, 64, 40),
       ([0] * 40 + [500] + [0] * 23, 0, 520, 522), ([5, 9], 2, 9, 11), ([3, 2, 2], 1, 1001, 13), ([1] * 64, 0, 8, 8), ([0, 0, 0], 0, 2050, 9), ([7] * 30, 0, 1030, 258),
       ([64, 65, 256, 257, 31, 0], 5, 1288, 1000), ([3] * 30 + [300, 0, 257, 256] + [1] * 36 + [64, 0, 65, 400], 1, 520, 264), ([150, 90], 0, 77, 65)]


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("counts,spare,k,n", FEW, ids=[f"{sum(c)}+{s}of{len(c)}-{k}x{n}" for c, s, k, n in FEW])
def test_weights_gradients_of_few_rows(counts, spare, k, n, dtype):
    g = torch.Generator().manual_seed(k * 7 + n)
    rows, held = sum(counts) + spare, sum(counts)
    x, dy = ((torch.randn(*s, generator=g)).to(dtype).cuda() for s in ((rows, k + 3), (rows, n + 5)))
    x[held:], dy[held:] = float("nan"), float("inf")        # nobody's
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    w = torch.empty(len(counts), n, k, dtype=dtype, device="cuda")
    for a, b in ((x[:, :k].contiguous(), dy[:, :n].contiguous()), (x[:, 3:], dy[:, 5:])):
        dw = hip_ops.expert_linear_backward(b, a, w, torch.from_numpy(offsets).cuda(), False, True)[1]
        za, zb = n64(a)[:held], n64(b)[:held]
        want, terms = (np.stack([f(zb[lo:hi]).T @ f(za[lo:hi]) for lo, hi in zip(offsets[:-1], offsets[1:])]) for f in (lambda v: v, np.abs))
        near(dw, want, terms, max(counts), dtype)


E4M3 = [([1], 0, 16, 1), ([0], 2, 16, 8), ([3, 0, 2, 1], 4, 128, 96), ([16, 1, 0, 33, 7], 0, 272, 72), ([40, 9], 2, 1008, 100), ([200, 0, 57, 130], 11, 320, 264), ([700, 0, 900], 5, 512, 768),
        ([2100, 1500], 0, 256, 513), ([5] * 70, 1, 64, 32), ([300, 300], 7, 144, 520), ([33, 100], 0, 16, 8), ([90], 0, 2048, 300), ([3001, 0, 1200], 7, 400, 8000), ([4200], 0, 1296, 7900)]


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("counts,spare,k,n", E4M3, ids=[f"{sum(c)}+{s}of{len(c)}-{k}x{n}" for c, s, k, n in E4M3])
def test_products_of_rows_in_8_bits(counts, spare, k, n, dtype):
    g = torch.Generator().manual_seed(k * 5 + n)
    rows, held = sum(counts) + spare, sum(counts)
    x, xs = nn.quantize_rows(torch.randn(rows, k, generator=g).cuda())
    w, ws = nn.quantize_rows(torch.randn(len(counts), n, k, generator=g).cuda())
    offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    y = nn.expert_linear_shard(x, w, torch.from_numpy(offsets).cuda(), x_scales=xs, weight_scales=ws, dtype=dtype)
    zx, zw = n64(x.float()) * n64(xs)[:, None], n64(w.float()) * n64(ws)[..., None]
    zx[held:] = 0
    near(y, o.product(zx, zw, offsets), o.product(np.abs(zx), np.abs(zw), offsets), k, dtype, IN_EIGHTS)


def test_strided_rows_and_one_gradient():
    g = torch.Generator().manual_seed(2)
    offsets = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")
    for dtype in DTYPES.values():
        big, w, dy = torch.randn(50, 200, generator=g).to(dtype).cuda(), torch.randn(2, 40, 64, generator=g).to(dtype).cuda(), torch.randn(50, 90, generator=g).to(dtype).cuda()
        for x, d in ((big[:, 8:72], dy[:, 16:56]), (big[:, 5:69], dy[:, 3:43])):
            want, terms = o.product(n64(x), n64(w), [0, 20, 50], n64(d)), o.product(np.abs(n64(x)), np.abs(n64(w)), [0, 20, 50], np.abs(n64(d)))
            a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
            near(nn.expert_linear_shard(x, w, offsets), want[0], terms[0], 64, dtype)
            near(torch.autograd.grad(nn.expert_linear_shard(a, w, offsets), [a], d)[0], want[1], terms[1], 40, dtype)
            near(torch.autograd.grad(nn.expert_linear_shard(x, b, offsets), [b], d)[0], want[2], terms[2], 30, dtype)


def test_rows_in_8_bits_that_lie_anywhere():
    """Rows and weights off 16 bytes and with pitches of their own are copied."""
    g = torch.Generator().manual_seed(6)
    offsets = torch.tensor([0, 20, 50], dtype=torch.int32, device="cuda")
    big, w = torch.randn(50, 100, generator=g).to(torch.float8_e4m3fn).cuda(), torch.randn(2 * 24 * 48 + 3, generator=g).to(torch.float8_e4m3fn).cuda()
    xs, ws = torch.rand(100, generator=g).cuda()[::2], torch.rand(2, 24, generator=g).cuda()
    for x, v in ((big[:, :48], w[:-3].view(2, 24, 48)), (big[:, 5:53], w[3:].view(2, 24, 48)), (big[:, 16:64], w[:-3].view(2, 24, 48))):
        y = nn.expert_linear_shard(x, v, offsets, x_scales=xs, weight_scales=ws, dtype=torch.float32)
        zx, zw = n64(x.float()) * n64(xs)[:, None], n64(v.float()) * n64(ws)[..., None]
        near(y, o.product(zx, zw, [0, 20, 50]), o.product(np.abs(zx), np.abs(zw), [0, 20, 50]), 48, torch.float32, IN_EIGHTS)


def test_offsets_that_hold_anything_stay_inside():
    """Whatever the offsets hold, rows of x, y and dw stay where they are; values outside 0 .. rows count as those."""
    x, w = torch.ones(40, 64, dtype=torch.bfloat16, device="cuda"), torch.ones(3, 32, 64, dtype=torch.bfloat16, device="cuda")
    offsets = torch.tensor([0, 10, 2 ** 31 - 1, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    assert (hip_ops.expert_linear(x, w, offsets) == 64).all()
    dx, dw = hip_ops.expert_linear_backward(torch.ones(40, 32, dtype=torch.bfloat16, device="cuda"), x, w, offsets)
    assert (dx == 32).all() and (dw[0] == 10).all() and (dw[1] == 30).all() and (dw[2] == 0).all()


def test_captured_and_replayed():
    g = torch.Generator().manual_seed(4)
    offsets = torch.tensor([0, 300, 300, 900], dtype=torch.int32, device="cuda")
    x, w, dy = ((torch.randn(*s, generator=g)).to(torch.bfloat16).cuda() for s in ((1000, 256), (3, 512, 256), (1000, 512)))

    def step():
        return (hip_ops.expert_linear(x, w, offsets),) + hip_ops.expert_linear_backward(dy, x, w, offsets)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for held in (1000, 17, 600):
        offsets.copy_(torch.tensor([0, held // 3, held // 2, held], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step()))


def test_a_feed_forward_block_of_experts():
    """Norm, routing, sort, two products with an activation between, combine: the gradients of the whole against torch in 64 bits; and its 8-bit form."""
    tokens, cols, hidden, experts, chosen = 90, 48, 80, 5, 2
    g = torch.Generator().manual_seed(11)

    def leaf(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=g)).cuda().requires_grad_()

    x, r, nw = leaf(tokens, cols), leaf(tokens, cols), leaf(cols)
    router, up, down = leaf(experts, cols, scale=0.3), leaf(experts, hidden, cols, scale=0.2), leaf(experts, cols, hidden, scale=0.2)

    h, stream = nn.rms_norm_shard(x, nw, r)
    top = (h @ router.t()).topk(chosen)
    weights = torch.softmax(top.values, -1)
    plan = nn.expert_plan(top.indices, experts)
    rows = nn.expert_sort(h, plan)
    out = stream + nn.expert_combine(nn.expert_linear_shard(torch.nn.functional.silu(nn.expert_linear_shard(rows, up, plan.offsets)), down, plan.offsets), plan, weights)
    dout = torch.randn(tokens, cols, generator=g).cuda()
    leaves = [x, r, nw, router, up, down]
    grads = torch.autograd.grad(out, leaves, dout)

    wide = [t.detach().double().requires_grad_() for t in leaves]
    x2, r2, nw2, router2, up2, down2 = wide
    s2 = x2 + r2
    h2 = s2 / torch.sqrt(s2.pow(2).mean(-1, keepdim=True) + 1e-6) * nw2
    w2 = torch.softmax((h2 @ router2.t()).gather(1, top.indices), -1)
    out2 = s2
    for j in range(chosen):
        a = torch.nn.functional.silu((up2[top.indices[:, j]] * h2[:, None]).sum(-1))
        out2 = out2 + w2[:, j:j + 1] * (down2[top.indices[:, j]] * a[:, None]).sum(-1)
    wants = torch.autograd.grad(out2, wide, dout.double())
    assert (out - out2).abs().max() < 1e-4
    for got, want in zip(grads, wants):
        assert (got - want).abs().max() <= 2e-5 * want.abs().max() + 1e-5

    with torch.no_grad():
        codes, scales, stream8 = nn.rms_norm_shard(x, nw, r, eight_bit=True)
        assert torch.equal(stream8, stream)
        rows8, row_scales = nn.expert_sort(codes, plan, scales)
        up8, up_scales = nn.quantize_rows(up)
        y8 = nn.expert_linear_shard(rows8, up8, plan.offsets, x_scales=row_scales, weight_scales=up_scales, dtype=torch.float32)
        y = nn.expert_linear_shard(rows, up, plan.offsets)
        # each factor is off by at most 2^-4 of itself, or 2^-10 of its row's scale: both together below 0.14 of the factors' sizes
        bound = 0.14 * torch.sqrt(rows.pow(2).sum(-1, keepdim=True)) * up.pow(2).sum(-1).sqrt().max()
        assert ((y8 - y).abs() <= bound).all()


def test_layers_over_workers_add_up():
    """Three workers with some of the experts each: what they combine adds up to all experts' result, and their weights' gradients are the whole's, in any order of sums."""
    from distdl_amd.backends.stub_hip import SimWorld
    tokens, cols, out, experts, chosen = 70, 40, 24, 7, 3
    g = torch.Generator().manual_seed(12)
    x, dy, w = torch.randn(tokens, cols, generator=g), torch.randn(tokens, out, generator=g), torch.randn(experts, out, cols, generator=g)
    ids, weights = torch.randint(0, experts, (tokens, chosen), generator=g), torch.rand(tokens, chosen, generator=g)

    def body(P_world, workers):
        P = P_world.create_partition_inclusive(list(range(workers))).create_cartesian_topology_partition([workers, 1])
        layer = nn.DistributedExpertLinear(P, experts, cols, out)
        assert layer.weight.shape[0] == layer.window[1] - layer.window[0]
        with torch.no_grad():
            layer.weight.copy_(w[slice(*layer.window)])
        a = x.cuda().requires_grad_()
        plan = nn.expert_plan(ids.cuda(), experts, window=layer.window)
        y = nn.expert_combine(layer(nn.expert_sort(a, plan), plan), plan, weights.cuda())
        y.backward(dy.cuda())
        return layer.window, n64(y), n64(a.grad), n64(layer.weight.grad)

    (whole,) = SimWorld(1).run(lambda P: body(P, 1))
    parts = SimWorld(3).run(lambda P: body(P, 3))
    assert [p[0] for p in parts] == [(0, 3), (3, 5), (5, 7)]
    for i in (1, 2):
        np.testing.assert_allclose(sum(p[i] for p in parts), whole[i], rtol=1e-5, atol=1e-4)
    np.testing.assert_allclose(np.concatenate([p[3] for p in parts]), whole[3], rtol=1e-5, atol=1e-4)
