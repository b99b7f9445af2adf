"""Gradients of fp32 weights from rows that lie beyond 2^31 bytes: what the forward pass takes, the adjoint takes."""

import pytest
import torch

from distdl_amd import _lib
from distdl_amd import nn

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def check(rows, pitch, bounds, n, k, at):
    """Every expert's gradient against 64 bits: sums of its rows' products in 32 bits, in any order."""
    g = torch.Generator(device="cuda").manual_seed(n)
    x = torch.empty(rows, pitch, device="cuda")
    x[:, at:at + k].normal_(generator=g)
    x = x[:, at:at + k]
    dy = torch.randn(rows, n, generator=g, device="cuda")
    w = torch.randn(len(bounds) - 1, n, k, generator=g, device="cuda").requires_grad_()
    offsets = torch.tensor(bounds, dtype=torch.int32, device="cuda")
    y = nn.expert_linear_shard(x, w, offsets)
    (dw,) = torch.autograd.grad(y, [w], dy)
    for e, (low, high) in enumerate(zip(bounds[:-1], bounds[1:])):
        want, terms = torch.zeros(n, k, dtype=torch.float64, device="cuda"), torch.zeros(n, k, dtype=torch.float64, device="cuda")
        for r in range(low, high, 8192):
            a, b = dy[r:min(r + 8192, high)].t().double().contiguous(), x[r:min(r + 8192, high)].double()
            want += torch.mm(a, b)
            terms += torch.mm(a.abs(), b.abs())
        assert ((dw[e] - want).abs() <= (2 * (high - low + 2) + 1) * U * terms).all()


@pytest.mark.parametrize("rows,pitch,bounds,n,k,at", [
    (66000, 8192, [0, 40, 30000, 30000, 65990], 24, 8192, 0),          # many rows
    (9000, 65536, [0, 5000, 8999], 96, 200, 65336),                    # far from each other, the last one at the end of its memory
    (640, 1 << 20, [0, 3, 40, 40, 70, 100, 639], 72, 40, 1001),        # the last expert's alone are many
    (600, 1 << 20, list(range(0, 601, 30)), 512, 320, 0),               # few for each expert
    (70000, 8191, [0, 70000], 5, 8191, 0)], ids=["rows", "pitch", "one", "few", "odd"])
def test_weights_gradients_of_far_rows(rows, pitch, bounds, n, k, at):
    check(rows, pitch, bounds, n, k, at)


def test_the_entry_point_with_32_bit_offsets_still_refuses():
    assert _lib.load().ddl_expert_linear_backward(16, 16, 16, _lib.DDL_DT_F32, 16, 2, 1 << 24, 64, 64, 64, 64, 16, 16, None) == -5
