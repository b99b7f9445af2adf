"""Root-mean-square norm, its residual, its 8-bit rows and its adjoint against the 64-bit oracle."""

import numpy as np
import pytest
import torch

from distdl_amd import hip_ops
from distdl_amd import nn
from oracle import experts as o

pytestmark = pytest.mark.gpu

U = 2.0 ** -24          # half a step of float32
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def half(dtype):
    return torch.finfo(dtype).eps / 2


def n64(t):
    return t.detach().double().cpu().numpy()


def make(g, dtype, *shape, scale=1.0):
    return (scale * torch.randn(*shape, generator=g)).to(dtype).cuda()


def check_rows(y, h, weight, eps, dtype):
    """A row's sum of squares is off by at most 40 roundings (16 elements a thread, ten levels of threads, and the squares), its root by half
    of that; four more roundings, and the result's."""
    want = o.rms_norm(n64(h), None if weight is None else n64(weight).reshape(-1), eps)[0]
    off = np.abs(n64(y) - want)
    assert (off <= (half(dtype) + 30 * U) * np.abs(want) + torch.finfo(dtype).tiny * (2.0 ** -10 if dtype != torch.float32 else 1)).all(), off.max()


SIZES = [(1, 1), (3, 7), (5, 8), (4, 9), (2, 63), (65, 64), (7, 100), (33, 511), (9, 512), (6, 513), (3, 1000), (17, 1024), (5, 1025), (3, 2048), (4, 2501),
         (2, 4096), (3, 5000), (2, 8191), (3, 8192), (2, 8200), (1, 16384), (2, 16383), (2050, 40)]


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_norm_and_adjoint(rows, cols, dtype):
    g = torch.Generator().manual_seed(rows * 31 + cols)
    x, r, dy, dh = (make(g, dtype, rows, cols) for _ in range(4))
    w = (1 + 0.3 * torch.randn(cols, generator=g)).to(dtype).cuda()
    for t in (x, r, w):
        t.requires_grad_()
    y, h = nn.rms_norm_shard(x, w, r, eps=1e-5)
    assert torch.equal(h, (x + r).detach())       # one rounding of the same sum
    check_rows(y, h, w, 1e-5, dtype)
    dx, dr, dw = torch.autograd.grad([y, h], [x, r, w], [dy, dh])
    assert torch.equal(dx, dr)
    want_dx, want_dw = o.rms_norm_backward(n64(dy), n64(h), n64(w), n64(dh), 1e-5)
    _, xhat, rstd = o.rms_norm(n64(h), None, 1e-5)
    gw = np.abs(n64(dy) * n64(w))
    size = rstd * (gw + np.abs(xhat) * (gw * np.abs(xhat)).mean(-1, keepdims=True)) + np.abs(n64(dh))
    assert (np.abs(n64(dx) - want_dx) <= half(dtype) * np.abs(want_dx) + 80 * U * size + 2.0 ** -25).all()
    terms = np.abs(n64(dy) * xhat).sum(0)
    assert (np.abs(n64(dw) - want_dw) <= half(dtype) * np.abs(want_dw) + (rows + 60) * U * terms + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("rows,cols,residual", [(1, 1, False), (3, 7, True), (5, 8, False), (4, 100, True), (33, 511, True), (3, 1000, False), (5, 1025, True),
                                                (2, 4096, True), (3, 8191, False), (16, 8192, True), (2, 16384, True)])
def test_rows_in_8_bits(rows, cols, residual, dtype):
    g = torch.Generator().manual_seed(rows * 37 + cols)
    x, w = make(g, dtype, rows, cols, scale=3), (1 + 0.3 * torch.randn(cols, generator=g)).to(dtype).cuda()
    r = make(g, dtype, rows, cols) if residual else None
    out = nn.rms_norm_shard(x, w, r, eight_bit=True)
    h = x if r is None else out[2]
    assert r is None or torch.equal(h, x + r)
    for codes, scales, y in ((out[0], out[1], o.rms_norm(n64(h), n64(w))[0]), nn.quantize_rows(x) + (n64(x),)):
        assert codes.dtype == torch.float8_e4m3fn and codes.shape == x.shape and scales.shape == x.shape[:1]
        want = o.row_scales(y)
        assert (np.abs(n64(scales) - want) <= 40 * U * want).all()
        # half a step of three mantissa bits, of 2^-9 below 2^-6, and what y and the scale are off themselves
        stands_for = codes.float().double().cpu().numpy() * n64(scales)[:, None]
        assert (np.abs(stands_for - y) <= (2.0 ** -4 + 100 * U) * np.abs(y) + (2.0 ** -10 + 100 * U) * n64(scales)[:, None]).all()


def test_rows_in_8_bits_at_the_ends():
    x = torch.zeros(6, 40, device="cuda")
    x[1, 3] = 1e-30
    x[2] = 3e38
    x[3, 5], x[4, 7] = float("inf"), float("nan")
    x[5, 0], x[5, 1] = 448.0, -1.75
    codes, scales = nn.quantize_rows(x)
    v = codes.float() * scales[:, None]
    assert (v[0] == 0).all() and scales[0] == 2.0 ** -126
    assert abs(v[1, 3] / 1e-30 - 1) < 1e-6 and (v[1, :3] == 0).all()
    assert (v[2] / 3e38 - 1).abs().max() < 1e-6
    assert v[3].isnan().all() and v[4, 7].isnan() and (v[4, :7] == 0).all()
    assert scales[5] == 1 and v[5, 0] == 448 and v[5, 1] == -1.75


def test_strided_rows_views_and_no_weight():
    g = torch.Generator().manual_seed(5)
    big = make(g, torch.bfloat16, 6, 3, 150)
    x, r = big[..., 10:110], big[..., 40:140]
    y, h = nn.rms_norm_shard(x, None, r)
    assert y.shape == x.shape and torch.equal(h, x + r)
    check_rows(y, h, None, 1e-6, torch.bfloat16)
    t = make(g, torch.float32, 40, 12).t()           # a stride in the columns
    check_rows(nn.rms_norm_shard(t), t, None, 1e-6, torch.float32)
    odd = make(g, torch.float16, 5 * 33 + 1)[1:].view(5, 33)      # off 16 bytes
    check_rows(nn.rms_norm_shard(odd), odd, None, 1e-6, torch.float16)
    assert nn.rms_norm_shard(x[:0]).shape == (0, 3, 100)
    w = torch.ones(100, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    (nn.rms_norm_shard(x[:0], w).sum()).backward()
    assert (w.grad == 0).all()


def test_gradients_of_one_result_alone_and_repeats():
    g = torch.Generator().manual_seed(6)
    x, r = make(g, torch.float32, 9, 130).requires_grad_(), make(g, torch.float32, 9, 130).requires_grad_()
    w = torch.ones(130, device="cuda", requires_grad=True)
    dh = make(g, torch.float32, 9, 130)
    y, h = nn.rms_norm_shard(x, w, r)
    dx, dr, dw = torch.autograd.grad(h, [x, r, w], dh, retain_graph=True)
    assert torch.equal(dx, dh) and torch.equal(dr, dh) and (dw == 0).all()
    one = torch.autograd.grad(y, [x, w], dh, retain_graph=True)
    two = torch.autograd.grad(y, [x, w], dh)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    want, want_w = o.rms_norm_backward(n64(dh), n64(h), n64(w))
    np.testing.assert_allclose(n64(one[0]), want, rtol=1e-4, atol=1e-5)
    np.testing.assert_allclose(n64(one[1]), want_w, rtol=1e-4, atol=1e-5)


def test_gradient_against_differences():
    g = torch.Generator().manual_seed(7)
    x, r = torch.randn(3, 20, generator=g, dtype=torch.float64), torch.randn(3, 20, generator=g, dtype=torch.float64)
    w, dy, dh = torch.randn(20, generator=g, dtype=torch.float64), torch.randn(3, 20, generator=g, dtype=torch.float64), torch.randn(3, 20, generator=g, dtype=torch.float64)

    def value(x):
        h = x.numpy() + r.numpy()
        return (o.rms_norm(h, w.numpy())[0] * dy.numpy()).sum() + (h * dh.numpy()).sum()

    leaf = x.float().cuda().requires_grad_()
    out = nn.rms_norm_shard(leaf, w.float().cuda(), r.float().cuda())
    (dx,) = torch.autograd.grad(out, [leaf], [dy.float().cuda(), dh.float().cuda()])
    for i in range(0, 60, 7):
        step = torch.zeros(60, dtype=torch.float64)
        step[i] = 1e-5
        slope = (value(x + step.view(3, 20)) - value(x - step.view(3, 20))) / 2e-5
        assert abs(slope - dx.view(-1)[i].item()) < 1e-4 * max(1, abs(slope))


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
def test_columns_spread_over_workers(dtype):
    """What two workers' launches leave and take, with unequal shares."""
    g = torch.Generator().manual_seed(8)
    x, r, dy, dh = (make(g, dtype, 11, 300) for _ in range(4))
    w = (1 + 0.3 * torch.randn(300, generator=g)).to(dtype).cuda()
    parts = [slice(0, 130), slice(130, 300)]
    first = [hip_ops.rms_norm(x[:, p], None, r[:, p], 1e-6, own_squares=True) for p in parts]
    squares = torch.stack([f[0] for f in first])
    y = torch.cat([hip_ops.rms_norm(f[1], w[p].contiguous(), None, 1e-6, part_squares=squares, total_cols=300)[0] for f, p in zip(first, parts)], 1)
    h = torch.cat([f[1] for f in first], 1)
    check_rows(y, h, w, 1e-6, dtype)
    sums = torch.stack([hip_ops.rms_norm_backward(dy[:, p], f[1], w[p].contiguous(), own_sums=True) for f, p in zip(first, parts)])
    grads = [hip_ops.rms_norm_backward(dy[:, p], f[1], w[p].contiguous(), dh[:, p], part_squares=squares, part_sums=sums, total_cols=300) for f, p in zip(first, parts)]
    want_dx, want_dw = o.rms_norm_backward(n64(dy), n64(h), n64(w), n64(dh))
    tol = 4 * half(dtype) + 1e-5
    np.testing.assert_allclose(np.concatenate([n64(a) for a, _ in grads], 1), want_dx, rtol=tol, atol=tol)
    np.testing.assert_allclose(np.concatenate([n64(b) for _, b in grads]), want_dw, rtol=tol, atol=tol)


def test_captured_and_replayed_on_another_stream():
    g = torch.Generator().manual_seed(9)
    x, r, dy, dh = (make(g, torch.bfloat16, 64, 1024) for _ in range(4))
    w = (1 + 0.3 * torch.randn(1024, generator=g)).to(torch.bfloat16).cuda()

    def step():
        h = hip_ops.rms_norm(x, w, r)
        return h[:2] + hip_ops.rms_norm_backward(dy, h[1], w, dh) + hip_ops.rms_norm(x, w, r, eight_bit=True)[1:]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for seed in range(3):
        x.copy_(make(torch.Generator().manual_seed(seed), torch.bfloat16, 64, 1024))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, step()):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


@pytest.mark.parametrize("shape,dims", [((2, 1, 2), 1), ((1, 2, 2), 2), ((2, 2, 1), 1), ((4, 1, 1), 2)])
def test_layer_over_four_workers(shape, dims):
    """Rows, columns or both on several workers: results and gradients of the whole tensor, the weight's summed over all rows."""
    from distdl_amd.backends.stub_hip import SimWorld
    from distdl_amd.utilities.slicing import compute_start_index, compute_subshape
    size = (5, 6, 10)
    g = torch.Generator().manual_seed(14)
    x, r, dy, dh = (torch.randn(*size, generator=g) for _ in range(4))
    w = 1 + 0.3 * torch.randn(*size[3 - dims:], generator=g)

    def body(P_world):
        P = P_world.create_partition_inclusive([0, 1, 2, 3]).create_cartesian_topology_partition(list(shape))
        layer = nn.DistributedRMSNorm(P, size[3 - dims:], eps=1e-5)
        start, extent = compute_start_index(shape, P.index, size), compute_subshape(shape, P.index, size)
        own = tuple(slice(int(s), int(s + e)) for s, e in zip(start, extent))
        if layer.weight.numel():
            with torch.no_grad():
                layer.weight.copy_(w[own[3 - dims:]].view(layer.weight.shape))
        a, b = x[own].cuda().requires_grad_(), r[own].cuda().requires_grad_()
        y, h = layer(a, b)
        torch.autograd.backward([y, h], [dy[own].cuda(), dh[own].cuda()])
        assert torch.equal(a.grad, b.grad)
        return own, n64(y), n64(h), n64(a.grad), None if layer.weight.grad is None else n64(layer.weight.grad)

    flat = (-1, int(np.prod(size[3 - dims:])))
    h = (x + r).double().numpy().reshape(flat)
    want = o.rms_norm(h, w.double().numpy().reshape(-1), 1e-5)[0].reshape(size)
    want_dx, want_dw = o.rms_norm_backward(dy.double().numpy().reshape(flat), h, w.double().numpy().reshape(-1), dh.double().numpy().reshape(flat), 1e-5)
    want_dx, want_dw = want_dx.reshape(size), want_dw.reshape(size[3 - dims:])
    for own, y, hh, dx, dw in SimWorld(4).run(body):
        np.testing.assert_allclose(y, want[own], rtol=1e-5, atol=1e-5)
        np.testing.assert_allclose(hh, h.reshape(size)[own], rtol=1e-6, atol=1e-6)
        np.testing.assert_allclose(dx, want_dx[own], rtol=1e-5, atol=1e-5)
        if dw is not None and dw.size:
            np.testing.assert_allclose(dw.reshape(want_dw[own[3 - dims:]].shape), want_dw[own[3 - dims:]], rtol=1e-4, atol=1e-4)


@pytest.mark.parametrize("eight_bit", [False, True])
def test_layer_without_rows(eight_bit):
    """No row of several dimensions is no row, not an unknown number of columns; a residual of another shape is refused, also where its elements would be enough."""
    from distdl_amd.backends.stub_hip import SimWorld

    def body(P_world):
        P = P_world.create_partition_inclusive([0]).create_cartesian_topology_partition([1, 1, 1])
        layer = nn.DistributedRMSNorm(P, (4, 8))
        x = torch.zeros(0, 4, 8, device="cuda")
        with torch.no_grad():
            res = layer(x, x.clone(), eight_bit=eight_bit)
            with pytest.raises(ValueError, match="residual"):
                layer(torch.zeros(3, 4, 8, device="cuda"), torch.zeros(3, 8, 4, device="cuda"), eight_bit=eight_bit)
        return [tuple(t.shape) for t in res]

    assert SimWorld(1).run(body)[0] == ([(0, 4, 8), (0,), (0, 4, 8)] if eight_bit else [(0, 4, 8)] * 2)
