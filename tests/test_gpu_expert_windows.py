"""The experts' products of some of the experts in the order: rows in front of theirs and behind them belong to none and become zeros, whatever the memory held."""

import numpy as np
import pytest
import torch

from distdl_amd import _lib
from distdl_amd import hip_ops
from distdl_amd import nn
from oracle import experts as o

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
CODES = {torch.float32: _lib.DDL_DT_F32, torch.bfloat16: _lib.DDL_DT_BF16, torch.float16: _lib.DDL_DT_F16}
# front, counts, spare, in, out: few rows by either kernel for them, tiles of every size
CASES = [(1, [1], 0, 16, 8), (3, [2, 0, 1], 1, 64, 40), (5, [0, 0], 0, 72, 33), (7, [], 2, 16, 9), (40, [9, 0, 16], 3, 264, 72), (17, [30] * 8, 2, 260, 1000),
         (33, [200, 57, 130], 11, 320, 264), (100, [2100, 1500], 0, 256, 512), (257, [3001, 1200], 7, 72, 8000), (260, [3001, 1200], 7, 8000, 72), (130, [400, 700], 0, 2050, 2049),
         (6, [100, 37], 3, 77, 65)]
IDS = [f"{f}+{sum(c)}+{s}of{len(c)}-{k}x{n}" for f, c, s, k, n in CASES]


def n64(t):
    return t.detach().double().cpu().numpy()


def near(got, want, terms, depth, dtype, more=0.0):
    """A sum of ``depth`` products in 32 bits, in any order, and the result's rounding (the smallest steps of fp16 aside)."""
    off = np.abs(n64(got) - want)
    assert (off <= torch.finfo(dtype).eps / 2 * np.abs(want) + (2 * (depth + 2) * U + more) * terms + 2.0 ** -25).all()


def operands(front, counts, spare, k, n, dtype):
    g = torch.Generator().manual_seed(k + n)
    rows, held = front + sum(counts) + spare, front + sum(counts)
    x, w, dy = (torch.randn(*s, generator=g).to(dtype).cuda() for s in ((rows, k), (len(counts), n, k), (rows, n)))
    x[:front], dy[:front], x[held:], dy[held:] = float("nan"), float("inf"), float("inf"), float("nan")        # nobody's
    offsets = (front + np.concatenate([[0], np.cumsum(counts)])).astype(np.int32)
    zx, zdy = n64(x), n64(dy)
    for z in (zx, zdy):
        z[:front], z[held:] = 0, 0
    return x, w, dy, torch.from_numpy(offsets).cuda(), zx, zdy


@pytest.mark.parametrize("dtype", CODES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("front,counts,spare,k,n", CASES, ids=IDS)
def test_rows_of_no_expert_become_zeros(front, counts, spare, k, n, dtype):
    x, w, dy, offsets, zx, zdy = operands(front, counts, spare, k, n, dtype)
    rows, lib, stream = x.shape[0], _lib.load(), hip_ops._stream()
    y, dx = (torch.full((rows, c), float("nan"), dtype=dtype, device="cuda") for c in (n, k))
    _lib.check(lib.ddl_expert_linear(x.data_ptr(), w.data_ptr(), CODES[dtype], offsets.data_ptr(), len(counts), rows, n, k, k, y.data_ptr(), stream), "forward")
    _lib.check(lib.ddl_expert_linear_backward(dy.data_ptr(), x.data_ptr(), w.data_ptr(), CODES[dtype], offsets.data_ptr(), len(counts), rows, n, k, n, k, dx.data_ptr(), None, stream),
               "adjoint")
    held = slice(front, front + sum(counts))
    for t in (y, dx):
        assert (t[:held.start] == 0).all() and (t[held.stop:] == 0).all()
    at = offsets.cpu().numpy()
    want, terms = o.product(zx, n64(w), at, zdy), o.product(np.abs(zx), np.abs(n64(w)), at, np.abs(zdy))
    near(y, want[0], terms[0], k, dtype)
    near(dx, want[1], terms[1], n, dtype)
    if counts:
        near(hip_ops.expert_linear_backward(dy, x, w, offsets, False, True)[1], want[2], terms[2], max(counts), dtype)


@pytest.mark.parametrize("dtype", CODES, ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("front,counts,spare,k,n", [(3, [2, 0, 1], 1, 64, 41), (7, [], 2, 16, 9), (17, [16, 1, 0, 33, 7], 0, 272, 72), (33, [200, 0, 57, 130], 11, 320, 264),
                                                    (60, [700, 0, 900], 5, 512, 768), (300, [3001, 0, 1200], 7, 400, 8000)])
def test_rows_in_8_bits_of_no_expert_become_zeros(front, counts, spare, k, n, dtype):
    g = torch.Generator().manual_seed(k * 5 + n)
    rows, held = front + sum(counts) + spare, slice(front, front + sum(counts))
    x, xs = nn.quantize_rows(torch.randn(rows, k, generator=g).cuda())
    w, ws = nn.quantize_rows(torch.randn(len(counts), n, k, generator=g).cuda())
    offsets = (front + np.concatenate([[0], np.cumsum(counts)])).astype(np.int32)
    there = torch.from_numpy(offsets).cuda()
    y = torch.full((rows, n), float("nan"), dtype=dtype, device="cuda")
    _lib.check(_lib.load().ddl_expert_linear_8bit(x.data_ptr(), xs.data_ptr(), w.data_ptr(), ws.data_ptr(), there.data_ptr(), len(counts), rows, n, k, k, y.data_ptr(),
                                                  CODES[dtype], hip_ops._stream()), "8 bits")
    assert (y[:held.start] == 0).all() and (y[held.stop:] == 0).all()
    zx, zw = n64(x.float()) * n64(xs)[:, None], n64(w.float()) * n64(ws)[..., None]
    # the matrix cores add eights, whose members they cut off at 2^-13 of the largest
    near(y, o.product(zx, zw, offsets), o.product(np.abs(zx), np.abs(zw), offsets), k, dtype, 7 * 2.0 ** -13)


def test_parts_of_a_plan_add_up():
    """The experts in two calls, with the parts of the plan's offsets and of the weights that go together: results and gradients of the rows add up to those of one call."""
    g = torch.Generator().manual_seed(5)
    plan = nn.expert_plan(torch.randint(0, 6, (200, 2), generator=g).cuda(), 6)
    x, w, dy = (torch.randint(-4, 5, s, generator=g).float().cuda() for s in ((400, 64), (6, 40, 64), (400, 40)))      # sums of whole numbers are exact
    def passes(lo, hi):
        a, b = x.clone().requires_grad_(), w[lo:hi].clone().requires_grad_()
        y = nn.expert_linear_shard(a, b, plan.offsets[lo:hi + 1])
        return (y.detach(),) + torch.autograd.grad(y, [a, b], dy)
    whole, low, high = passes(0, 6), passes(0, 4), passes(4, 6)
    for i in (0, 1):
        assert torch.equal(low[i] + high[i], whole[i])
    assert torch.equal(torch.cat([low[2], high[2]]), whole[2])
