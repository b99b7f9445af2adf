"""Refusals and host logic of the experts' operators; no GPU."""

import numpy as np
import pytest
import torch

from distdl_amd import _lib
from distdl_amd import nn
from oracle import experts as o

BF16, F32, F64 = _lib.DDL_DT_BF16, _lib.DDL_DT_F32, _lib.DDL_DT_F64


def call(name, defaults, change):
    assert set(change) <= set(defaults)
    return getattr(_lib.load(), name)(*{**defaults, **change}.values())


def refused(name, defaults, change, code, what):
    assert call(name, defaults, change) == code
    assert what in _lib.load().ddl_last_error().decode()


NORM = dict(x=16, residual=None, weight=None, dtype=BF16, rows=4, cols=64, ld_x=64, ld_r=0, eps=1e-6, sum=None, y=16, codes=None, scales=None, own=None,
            parts=None, nparts=0, total=64, stream=None)


@pytest.mark.parametrize("change,code,what", [
    (dict(dtype=F64), -1, "dtype"), (dict(rows=-1), -1, "rows"), (dict(cols=0), -1, "columns"), (dict(cols=16385, ld_x=16385), -5, "16384"), (dict(eps=-1.0), -1, "eps"),
    (dict(eps=float("nan")), -1, "eps"), (dict(x=None), -1, "null"), (dict(y=None), -1, "null"), (dict(residual=16, ld_r=64), -1, "null"), (dict(ld_x=63), -1, "pitch"),
    (dict(residual=16, sum=16, ld_r=63), -1, "pitch"), (dict(codes=16), -1, "codes"), (dict(codes=16, y=None), -1, "codes"), (dict(codes=16, y=None, scales=16, own=16), -1, "codes"),
    (dict(own=16, parts=16, nparts=2), -1, "asked for"), (dict(parts=16), -1, "0 workers"), (dict(parts=16, nparts=2, total=60), -1, "of 60 columns"),
])
def test_norm_refuses(change, code, what):
    refused("ddl_rms_norm", NORM, change, code, what)


NORM_BACKWARD = dict(dy=16, h=16, dh=None, weight=16, dtype=BF16, rows=4, cols=64, ld_dy=64, ld_h=64, ld_dh=0, eps=1e-6, dx=16, dw=None, work=None, elems=0, own=None,
                     squares=None, sums=None, nparts=0, total=64, stream=None)


@pytest.mark.parametrize("change,code,what", [
    (dict(dtype=F64), -1, "dtype"), (dict(cols=20000), -5, "16384"), (dict(dw=16), -1, "workspace"), (dict(dw=16, work=16, elems=255), -1, "256 are needed"), (dict(dy=None), -1, "null"),
    (dict(ld_dy=60), -1, "pitch"), (dict(dh=16, ld_dh=60), -1, "pitch"), (dict(sums=16, nparts=2), -1, "squares"), (dict(own=16), -1, "or gradients"), (dict(eps=-1.0), -1, "eps"),
])
def test_norm_adjoint_refuses(change, code, what):
    refused("ddl_rms_norm_backward", NORM_BACKWARD, change, code, what)


PLAN = dict(ids=16, id_bytes=8, tokens=4, chosen=2, ld=2, low=0, high=8, place=16, offsets=16, work=None, elems=0, stream=None)


@pytest.mark.parametrize("change,code,what", [
    (dict(id_bytes=2), -1, "2 bytes"), (dict(tokens=-1), -1, "tokens"), (dict(high=-1), -1, "experts"), (dict(low=-1), -1, "experts"), (dict(high=2048), -5, "2047"),
    (dict(tokens=1 << 30), -5, "2^30"), (dict(offsets=None), -1, "null"), (dict(ids=None), -1, "null"), (dict(place=None), -1, "null"), (dict(tokens=4000), -1, "workspace"),
    (dict(tokens=4000, work=16, elems=143), -1, "144 are needed"),
])
def test_plan_refuses(change, code, what):
    refused("ddl_expert_plan", PLAN, change, code, what)


SORT = dict(x=16, bytes=2, tokens=4, chosen=2, cols=64, ld=64, place=16, held=16, out=16, scales=None, out_scales=None, stream=None)
COMBINE = dict(y=16, dtype=BF16, tokens=4, chosen=2, cols=64, ld=64, place=16, held=16, weights=None, out=16, stream=None)
COMBINE_BACKWARD = dict(dout=16, y=16, dtype=BF16, tokens=4, chosen=2, cols=64, ld_dout=64, ld_y=64, place=16, held=16, weights=16, dy=16, dweights=16, stream=None)


@pytest.mark.parametrize("name,defaults,change,code,what", [
    ("ddl_expert_sort", SORT, dict(bytes=8), -1, "8 bytes"), ("ddl_expert_sort", SORT, dict(cols=0), -1, "columns"), ("ddl_expert_sort", SORT, dict(ld=63), -1, "pitch"),
    ("ddl_expert_sort", SORT, dict(place=None), -1, "null"), ("ddl_expert_sort", SORT, dict(scales=16), -1, "null"), ("ddl_expert_sort", SORT, dict(tokens=1 << 31), -5, "2^30"),
    ("ddl_expert_sort", SORT, dict(tokens=1 << 28, cols=1 << 20, ld=1 << 20), -5, "wavefronts"),
    ("ddl_expert_combine", COMBINE, dict(dtype=F64), -1, "dtype"), ("ddl_expert_combine", COMBINE, dict(ld=60), -1, "pitch"), ("ddl_expert_combine", COMBINE, dict(y=None), -1, "null"),
    ("ddl_expert_combine", COMBINE, dict(held=None), -1, "null"), ("ddl_expert_combine", COMBINE, dict(chosen=-1), -1, "choices"),
    ("ddl_expert_combine_backward", COMBINE_BACKWARD, dict(weights=None), -1, "null"), ("ddl_expert_combine_backward", COMBINE_BACKWARD, dict(y=None), -1, "null"),
    ("ddl_expert_combine_backward", COMBINE_BACKWARD, dict(ld_y=1), -1, "pitch"), ("ddl_expert_combine_backward", COMBINE_BACKWARD, dict(dtype=0), -1, "dtype"),
])
def test_moves_refuse(name, defaults, change, code, what):
    refused(name, defaults, change, code, what)


LINEAR = dict(x=16, w=16, dtype=BF16, offsets=16, experts=2, rows=4, n=64, k=64, ld=64, y=16, stream=None)
LINEAR8 = dict(x=16, xs=16, w=16, ws=16, offsets=16, experts=2, rows=4, n=64, k=64, ld=64, y=16, dtype=BF16, stream=None)
LINEAR_BACKWARD = dict(dy=16, x=16, w=16, dtype=BF16, offsets=16, experts=2, rows=4, n=64, k=64, ld_dy=64, ld_x=64, dx=16, dw=16, stream=None)


@pytest.mark.parametrize("name,defaults,change,code,what", [
    ("ddl_expert_linear", LINEAR, dict(dtype=F64), -1, "dtype"), ("ddl_expert_linear", LINEAR, dict(k=7), -5, "at least 8"), ("ddl_expert_linear", LINEAR, dict(n=7), -5, "at least 8"),
    ("ddl_expert_linear", LINEAR, dict(n=0), -1, "features"), ("ddl_expert_linear", LINEAR, dict(rows=1 << 30), -5, "rows"), ("ddl_expert_linear", LINEAR, dict(experts=65535), -5, "experts"),
    ("ddl_expert_linear", LINEAR, dict(n=40000, k=40000, ld=40000), -5, "features"), ("ddl_expert_linear", LINEAR, dict(ld=63), -1, "pitch"), ("ddl_expert_linear", LINEAR, dict(ld=1 << 23), -5, "2^22"),
    ("ddl_expert_linear", LINEAR, dict(w=None), -1, "null"), ("ddl_expert_linear", LINEAR, dict(offsets=None), -1, "null"),
    ("ddl_expert_linear_8bit", LINEAR8, dict(k=24, ld=32), -3, "multiple of 16"), ("ddl_expert_linear_8bit", LINEAR8, dict(ld=72), -3, "16-byte"), ("ddl_expert_linear_8bit", LINEAR8, dict(x=24), -3, "16-byte"),
    ("ddl_expert_linear_8bit", LINEAR8, dict(dtype=F64), -1, "dtype"), ("ddl_expert_linear_8bit", LINEAR8, dict(ws=None), -1, "null"), ("ddl_expert_linear_8bit", LINEAR8, dict(rows=-1), -1, "rows"),
    ("ddl_expert_linear_backward", LINEAR_BACKWARD, dict(dtype=F64), -1, "dtype"), ("ddl_expert_linear_backward", LINEAR_BACKWARD, dict(ld_dy=60), -1, "pitch"),
    ("ddl_expert_linear_backward", LINEAR_BACKWARD, dict(ld_x=60), -1, "pitch"), ("ddl_expert_linear_backward", LINEAR_BACKWARD, dict(x=None), -1, "null"),
    ("ddl_expert_linear_backward", LINEAR_BACKWARD, dict(dtype=F32, rows=1 << 24), -5, "2^31"), ("ddl_expert_linear_backward", LINEAR_BACKWARD, dict(ld_dy=1 << 23), -5, "2^22"),
])
def test_products_refuse(name, defaults, change, code, what):
    refused(name, defaults, change, code, what)


def test_nothing_is_no_launch():
    assert call("ddl_rms_norm", NORM, dict(rows=0)) == 0
    assert call("ddl_rms_norm_backward", NORM_BACKWARD, dict(rows=0)) == 0
    assert call("ddl_expert_sort", SORT, dict(tokens=0)) == call("ddl_expert_sort", SORT, dict(chosen=0)) == 0
    assert call("ddl_expert_combine", COMBINE, dict(tokens=0)) == call("ddl_expert_combine_backward", COMBINE_BACKWARD, dict(tokens=0)) == 0
    assert call("ddl_expert_linear", LINEAR, dict(rows=0)) == call("ddl_expert_linear_8bit", LINEAR8, dict(rows=0)) == 0
    assert call("ddl_expert_linear_backward", LINEAR_BACKWARD, dict(rows=0, dw=None)) == 0


@pytest.mark.parametrize("extents", [(-1, 8), (1 << 40, 8), (5000, -1), (5000, 2048), (2048, 8)])
def test_plans_without_a_workspace(extents):
    assert _lib.load().ddl_expert_plan_workspace(*extents) == 0


@pytest.mark.parametrize("extents", [(-1, 8), (0, 8), (5, 0), (5, 20000)])
def test_norms_without_a_workspace(extents):
    assert _lib.load().ddl_rms_norm_backward_workspace(*extents) == 0


def test_tensors_off_the_gpu_are_refused():
    x, ids = torch.zeros(4, 16), torch.zeros(4, 2, dtype=torch.int64)
    plan = nn.ExpertPlan(torch.zeros(4, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), (0, 2))
    for f in (lambda: nn.rms_norm_shard(x), lambda: nn.rms_norm_shard(x, eight_bit=True), lambda: nn.quantize_rows(x), lambda: nn.expert_plan(ids, 4),
              lambda: nn.expert_sort(x, plan), lambda: nn.expert_combine(torch.zeros(8, 16), plan), lambda: nn.expert_linear_shard(x, torch.zeros(2, 8, 16), plan.offsets)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            f()


def test_rows_in_8_bits_have_no_gradient():
    x, s = torch.zeros(4, 16, requires_grad=True), torch.zeros(4, requires_grad=True)
    codes = torch.zeros(4, 16, dtype=torch.float8_e4m3fn)
    plan = nn.ExpertPlan(torch.zeros(4, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), (0, 2))
    for f in (lambda: nn.rms_norm_shard(x, eight_bit=True), lambda: nn.quantize_rows(x), lambda: nn.expert_sort(codes, plan, s),
              lambda: nn.expert_linear_shard(codes, torch.zeros(2, 8, 16, dtype=torch.float8_e4m3fn), plan.offsets, x_scales=s, weight_scales=torch.zeros(2, 8))):
        with pytest.raises(ValueError, match="no gradient"):
            f()


def test_arguments_of_plans_and_layers():
    from distdl_amd.backends.stub_hip import SimWorld
    ids = torch.zeros(4, 2, dtype=torch.int64)
    for bad in (dict(num_experts=-1), dict(num_experts=2.5), dict(num_experts=4, window=(2, 5)), dict(num_experts=4, window=(3, 2)), dict(num_experts=4, window=(-1, 2))):
        with pytest.raises(ValueError):
            nn.expert_plan(ids, **bad)
    for bad in (ids[0], ids.float(), ids.to(torch.int16)):
        with pytest.raises(ValueError, match="int32 or int64"):
            nn.expert_plan(bad, 4)
    P = SimWorld(2).partition(0).create_partition_inclusive([0, 1])
    with pytest.raises(ValueError, match="first dimension"):
        nn.DistributedExpertLinear(P.create_cartesian_topology_partition([1, 2]), 4, 8, 8, device="cpu")
    layer = nn.DistributedExpertLinear(P.create_cartesian_topology_partition([2, 1]), 5, 8, 16, device="cpu")
    assert layer.window == (0, 3) and layer.weight.shape == (3, 16, 8)
    with pytest.raises(ValueError, match="holds"):
        layer(torch.zeros(4, 8), nn.ExpertPlan(ids, ids, (3, 5)))
    norm = nn.DistributedRMSNorm(P.create_cartesian_topology_partition([1, 2]), 10, device="cpu")
    assert norm.weight.shape == (1, 5) and (norm.weight == 1).all()
    with pytest.raises(ValueError, match="gives this worker"):
        norm(torch.zeros(3, 10))
    with pytest.raises(ValueError, match="whole on their worker"):
        norm(torch.zeros(3, 5), eight_bit=True)
    with pytest.raises(ValueError, match="normalised dimensions"):
        nn.DistributedRMSNorm(P.create_cartesian_topology_partition([1, 2]), (1, 2, 3), device="cpu")
    with pytest.raises(ValueError, match="no elements"):
        nn.DistributedRMSNorm(P.create_cartesian_topology_partition([1, 2]), 1, device="cpu")


def test_the_oracle_against_torch():
    rng = np.random.default_rng(0)
    h, w, dy, dh = rng.standard_normal((5, 12)), rng.standard_normal(12), rng.standard_normal((5, 12)), rng.standard_normal((5, 12))
    t, tw = torch.tensor(h, requires_grad=True), torch.tensor(w, requires_grad=True)
    y = torch.nn.functional.rms_norm(t, (12,), tw, 1e-6)
    np.testing.assert_allclose(o.rms_norm(h, w)[0], y.detach().numpy(), rtol=1e-12)
    dx, dw = torch.autograd.grad([y, t], [t, tw], [torch.tensor(dy), torch.tensor(dh)])
    got = o.rms_norm_backward(dy, h, w, dh)
    np.testing.assert_allclose(got[0], dx.numpy(), rtol=1e-10, atol=1e-12)
    np.testing.assert_allclose(got[1], dw.numpy(), rtol=1e-10, atol=1e-12)
    ids = rng.integers(-1, 6, (9, 3))
    place, offsets = o.plan(ids, 1, 5)
    for e in range(1, 5):
        rows = [place[t, j] for t in range(9) for j in range(3) if ids[t, j] == e]
        assert rows == list(range(offsets[e - 1], offsets[e]))
    assert sorted(place.reshape(-1)) == list(range(27))
    x = rng.standard_normal((9, 4))
    weights = rng.random((9, 3))
    held = (ids >= 1) & (ids < 5)
    np.testing.assert_allclose(o.combine(o.sort(x, place, offsets[-1]), place, offsets[-1], weights), x * (weights * held).sum(1, keepdims=True), rtol=1e-12)
