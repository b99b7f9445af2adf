"""Tangents and traces that meet the experts' operators: they see the torch.autograd.Functions, so that nothing is dropped.  No GPU: the kernels' calls are
replaced by definitions in NumPy, which torch does not see either."""

import numpy as np
import pytest
import torch

from distdl_amd import hip_ops
from distdl_amd import nn
from oracle import experts as o


def _numpy(t):
    return t.detach().numpy()


def _rows8(y):
    scales = torch.from_numpy(o.row_scales(y).astype(np.float32))
    return (torch.from_numpy(np.asarray(y, np.float32)) / scales[..., None]).to(torch.float8_e4m3fn), scales


@pytest.fixture
def kernels(monkeypatch):
    def rms_norm(x, weight=None, residual=None, eps=1e-6, eight_bit=False):
        h = x if residual is None else x.detach() + residual.detach()
        y = o.rms_norm(_numpy(h), None if weight is None else _numpy(weight), eps)[0].astype(np.float32)
        return (None, h) + _rows8(y) if eight_bit else (torch.from_numpy(y), h, None, None)

    def expert_plan(ids, low, high):
        place, offsets = o.plan(_numpy(ids), low, high)
        return torch.from_numpy(place.astype(np.int32)), torch.from_numpy(offsets.astype(np.int32))

    def expert_sort(x, place, offsets, scales=None):
        rows = torch.from_numpy(o.sort(_numpy(x.float()), _numpy(place), int(offsets[-1])))
        return (rows.to(x.dtype), torch.from_numpy(o.sort(_numpy(scales)[:, None], _numpy(place), int(offsets[-1]))[:, 0])) if scales is not None else (rows, None)

    def expert_combine(y, place, offsets, weights=None):
        return torch.from_numpy(o.combine(_numpy(y), _numpy(place), int(offsets[-1]), None if weights is None else _numpy(weights)).astype(np.float32))

    def expert_linear(x, weight, offsets, x_scales=None, weight_scales=None, dtype=None):
        return torch.from_numpy(o.product(_numpy(x.float()), _numpy(weight.float()), _numpy(offsets)).astype(np.float32))

    for f in (rms_norm, expert_plan, expert_sort, expert_combine, expert_linear):
        monkeypatch.setattr(hip_ops, f.__name__, f)
    monkeypatch.setattr(hip_ops, "quantize_rows", lambda x: _rows8(_numpy(x)))


PLACE, OFFSETS = torch.tensor([[0, 2], [3, 1], [4, 5]], dtype=torch.int32), torch.tensor([0, 2, 5], dtype=torch.int32)
PLAN = nn.ExpertPlan(PLACE, OFFSETS, (0, 2))


def _operators():
    """Name: (call of one tensor, its shape, the name of its function)."""
    w, codes, ones = torch.randn(2, 5, 8), torch.randn(6, 8).to(torch.float8_e4m3fn), torch.ones(6)
    return {"norm": (lambda x: nn.rms_norm_shard(x, None), (3, 8), "_RmsNormShard"),
            "norm_residual": (lambda x: nn.rms_norm_shard(x, None, x)[0], (3, 8), "_RmsNormShard"),
            "norm_eight": (lambda x: nn.rms_norm_shard(x, eight_bit=True)[1], (3, 8), "_RmsNormEight"),
            "quantize": (lambda x: nn.quantize_rows(x)[1], (3, 8), "_QuantizeRows"),
            "sort": (lambda x: nn.expert_sort(x, PLAN), (3, 8), "_ExpertSort"),
            "sort_eight": (lambda s: nn.expert_sort(codes[:3], PLAN, s)[1], (3,), "_ExpertSortEight"),
            "combine": (lambda y: nn.expert_combine(y, PLAN), (6, 8), "_ExpertCombine"),
            "linear": (lambda x: nn.expert_linear_shard(x, w, OFFSETS), (6, 8), "_ExpertLinear"),
            "linear_eight": (lambda s: nn.expert_linear_shard(codes, w.to(torch.float8_e4m3fn), OFFSETS, x_scales=s, weight_scales=torch.ones(2, 5)), (6,), "_ExpertLinearEight")}


NAMES = ["norm", "norm_residual", "norm_eight", "quantize", "sort", "sort_eight", "combine", "linear", "linear_eight"]


@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("name", NAMES)
def test_tangents_are_not_dropped(kernels, name, grad_mode):
    call, shape, _ = _operators()[name]
    x = torch.rand(*shape) + 1
    with torch.set_grad_enabled(grad_mode), torch.autograd.forward_ad.dual_level():
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
            call(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("name", NAMES)
def test_traces_hold_the_call(kernels, name):
    call, shape, function = _operators()[name]
    first, second = torch.rand(*shape) + 1, torch.rand(*shape) + 2
    traced = torch.jit.trace(call, (first,), check_trace=False)
    assert function in str(traced.graph)
    assert torch.equal(traced(second), call(second))


@pytest.mark.filterwarnings("ignore")
def test_a_traced_plan_is_made_anew(kernels):
    def call(ids):
        plan = nn.expert_plan(ids, 4)
        return plan.place, plan.offsets
    traced = torch.jit.trace(call, (torch.tensor([[0, 1], [2, 3]]),), check_trace=False)
    ids = torch.tensor([[3, 3], [1, -1]])
    assert all(torch.equal(a, b) for a, b in zip(traced(ids), call(ids)))
    assert traced(ids)[1].tolist() == [0, 0, 1, 1, 3]


@pytest.mark.parametrize("name", ["norm", "sort", "combine", "linear"])
def test_calls_without_gradients_record_nothing(kernels, name):
    call, shape, _ = _operators()[name]
    x, leaf = torch.randn(*shape), torch.randn(*shape, requires_grad=True)
    assert not call(x).requires_grad and call(leaf).requires_grad
    with torch.no_grad():
        assert not call(leaf).requires_grad
