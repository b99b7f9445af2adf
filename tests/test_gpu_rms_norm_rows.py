"""Root-mean-square norm where a group of threads has some rows one after the other: every row is what it is as the first of its group, and the weight's gradient
is the sum over all of them."""

import numpy as np
import pytest
import torch

from distdl_amd import nn
from oracle import experts as o

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# Every kind of group (64 threads with one or two pieces of a row, 256, 512, 1024 with one or two) with rows of whole pieces and others, and two rows a group at least
SIZES = [(9000, 100), (8300, 512), (8400, 1000), (2100, 1025), (2300, 2048), (1100, 2501), (1300, 4096), (1100, 8191), (700, 8192), (1100, 9000)]


def n64(t):
    return t.detach().double().cpu().numpy()


def operands(rows, cols, dtype):
    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x, r, dy, dh = (torch.randn(rows, cols, generator=g, device="cuda").to(dtype) for _ in range(4))
    return x, r, (1 + 0.3 * torch.randn(cols, generator=g, device="cuda")).to(dtype), dy, dh


def results(x, r, w, dy, dh):
    leaves = [t.detach().clone().requires_grad_() for t in (x, r, w)]
    y, h = nn.rms_norm_shard(*[leaves[0], leaves[2], leaves[1]])
    dx, dr, dw = torch.autograd.grad([y, h], leaves, [dy, dh])
    alone = nn.rms_norm_shard(x, w)
    with torch.no_grad():
        codes, scales, h8 = nn.rms_norm_shard(x, w, r, eight_bit=True)
        plain, plain_scales = nn.quantize_rows(x)
    assert torch.equal(dx, dr) and torch.equal(h, h8)
    return [y, h, dx, alone, codes.view(torch.uint8), scales, plain.view(torch.uint8), plain_scales], dw


@pytest.mark.parametrize("dtype", DTYPES.values(), ids=DTYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_every_row_of_a_group(rows, cols, dtype):
    x, r, w, dy, dh = operands(rows, cols, dtype)
    many, dw = results(x, r, w, dy, dh)
    for first in range(0, rows, 500):
        part = slice(first, first + 500)      # as many rows as that are one a group
        few, _ = results(x[part], r[part], w, dy[part], dh[part])
        assert all(torch.equal(a[part], b) for a, b in zip(many, few))
    _, xhat, _ = o.rms_norm(n64(many[1]), None)
    terms, want = np.abs(n64(dy) * xhat).sum(0), (n64(dy) * xhat).sum(0)
    # sums of all rows in any order, the rows' own factor off by 30 roundings at most
    assert (np.abs(n64(dw) - want) <= torch.finfo(dtype).eps / 2 * np.abs(want) + (rows + 60) * U * terms + 2.0 ** -25).all()
    # what the groups' sums would lack or hold twice shows in rows of one sign
    ones = torch.ones_like(x)
    leaf = w.clone().requires_grad_()
    (count,) = torch.autograd.grad(nn.rms_norm_shard(ones, leaf, eps=0.0), [leaf], ones)
    assert (count == torch.tensor(rows, device="cuda").to(dtype)).all()
