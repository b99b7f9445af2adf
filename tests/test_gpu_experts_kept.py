"""What the way back keeps for its adjoint: the experts' rows for the router weights' gradient, and nothing of their size where that is not wanted."""

import numpy as np
import pytest
import torch

from distdl_amd import hip_ops
from distdl_amd import nn
from oracle import experts as o

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["native", "general"])
def path(request, monkeypatch):
    if request.param == "general":
        from distdl_amd import _lib

        class General:
            def __getattr__(self, _):
                return lambda *a: None

        monkeypatch.setattr(_lib, "front", General)


def _operands(dtype, wants_weights):
    g = torch.Generator().manual_seed(21)
    ids = torch.randint(-1, 5, (40, 3), generator=g)
    y = torch.randn(120, 24, generator=g).to(dtype).cuda().requires_grad_()
    weights = None if wants_weights is None else torch.rand(40, 3, generator=g).cuda().requires_grad_(wants_weights)
    return ids, y, weights, torch.randn(40, 24, generator=g).to(dtype).cuda()


def _kept(f):
    shapes = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: shapes.append(tuple(t.shape)) or t, lambda t: t):
        out = f()
    return out, shapes


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("weighted", [False, True], ids=["ones", "weights"])
def test_rows_may_change_where_no_gradient_needs_them(path, weighted, dtype):
    ids, y, weights, dout = _operands(dtype, False if weighted else None)
    plan = nn.expert_plan(ids.cuda(), 5, window=(1, 5))
    place, offsets = o.plan(ids.numpy(), 1, 5)
    assert (120, 24) not in _kept(lambda: nn.expert_combine(y, plan, weights))[1]
    out = nn.expert_combine(y, plan, weights)      # a tensor that hooks have packed has no version
    with torch.no_grad():
        y.fill_(float("nan"))
    (dy,) = torch.autograd.grad(out, [y], dout)
    held, ones = offsets[-1], np.ones((40, 3))
    want = o.combine_backward(dout.double().cpu().numpy(), np.zeros((120, 24)), place, held, weights.double().cpu().numpy() if weighted else ones)[0]
    got = dy.double().cpu().numpy()
    # one product, rounded once in 32 bits and once to the type
    assert (np.abs(got - want) <= (torch.finfo(dtype).eps / 2 + 2.0 ** -24) * np.abs(want)).all()


def test_rows_are_kept_for_the_weights(path):
    ids, y, weights, dout = _operands(torch.float32, True)
    plan = nn.expert_plan(ids.cuda(), 5, window=(1, 5))
    assert _kept(lambda: nn.expert_combine(y, plan, weights))[1].count((120, 24)) == 1
    out = nn.expert_combine(y, plan, weights)
    with torch.no_grad():
        y.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, [y], dout)


def test_the_adjoint_without_rows(path):
    ids, y, weights, dout = _operands(torch.float32, False)
    plan = nn.expert_plan(ids.cuda(), 5, window=(1, 5))
    both = hip_ops.expert_combine_backward(dout, y.detach(), plan.place, plan.offsets, weights)
    dy, none = hip_ops.expert_combine_backward(dout, None, plan.place, plan.offsets, weights, True, False)
    assert none is None and torch.equal(dy, both[0])
    with pytest.raises(ValueError, match="need the rows"):
        hip_ops.expert_combine_backward(dout, None, plan.place, plan.offsets, weights)
