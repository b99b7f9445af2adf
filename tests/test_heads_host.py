"""Refusals and host logic of the heads' operators; no GPU."""

import ctypes

import numpy as np
import pytest
import torch

from distdl_amd import _lib
from distdl_amd import hip_ops
from distdl_amd import nn
from oracle import heads as o_heads


def _i64(*v):
    return _lib.i64_array(v)


def _rotary(lib, **change):
    a = dict(q=1, qs=_i64(8, 8, 8), k=None, ks=None, dtype=_lib.DDL_DT_F32, batch=1, tokens=1, qh=1, kh=0, dim=8, qw=None, kw=None, norm=0, eps=1e-6,
             freq=1, rotated=8, pos=None, pos_bytes=0, pos_batch=0, neighbours=0, amplitude=1.0, inverse=0, yq=1, yqs=_i64(8, 8, 8), yk=None, yks=None,
             stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return lib.ddl_head_rotary(*a.values())


@pytest.mark.parametrize("change,code,what", [
    (dict(dtype=_lib.DDL_DT_F64), -1, "dtype"), (dict(batch=-1), -1, "negative"), (dict(dim=0), -1, "empty"), (dict(dim=520), -5, "at most 512"),
    (dict(rotated=7), -4, "pairs"), (dict(rotated=10), -4, "pairs"), (dict(freq=None), -1, "frequencies"), (dict(pos_bytes=2, pos=1), -1, "positions"),
    (dict(pos_bytes=8), -1, "positions"), (dict(q=None), -1, "null"), (dict(yqs=None), -1, "null"), (dict(qw=1), -1, "without a norm"),
    (dict(norm=1, inverse=1), -1, "adjoint"), (dict(batch=1 << 20, tokens=1 << 20), -5, "2^31"),
])
def test_rotation_refuses(change, code, what):
    lib = _lib.load()
    assert _rotary(lib, **change) == code
    assert what in lib.ddl_last_error().decode()


def test_rotation_of_nothing_is_no_launch():
    lib = _lib.load()
    assert _rotary(lib, tokens=0) == 0
    assert _rotary(lib, qh=0) == 0


def test_adjoint_of_head_norms_asks_for_its_workspace():
    lib = _lib.load()
    need = lib.ddl_head_norm_rotary_backward_workspace(64)
    assert need >= 128
    st = _i64(64, 64, 64)
    rc = lib.ddl_head_norm_rotary_backward(1, st, None, None, 1, st, None, None, _lib.DDL_DT_F32, 1, 1, 1, 0, 64, None, None, 1e-6, 1, 64, None, 0, 0, 0,
                                           1.0, 1, st, None, None, 1, None, None, need - 1, None)
    assert rc == -1 and "workspace" in lib.ddl_last_error().decode()


def test_tensors_off_the_gpu_are_refused():
    q, freq = torch.zeros(1, 1, 1, 8), nn.rotary_frequencies(8)
    for call in (lambda: nn.rotary_shard(q, None, freq), lambda: nn.head_norm_rotary_shard(q, None, None, None, freq)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


def test_frequencies_and_their_scalings():
    f = nn.rotary_frequencies(8, base=100.0).numpy()
    assert f.dtype == np.float64 and np.allclose(f, [1, 100 ** -0.25, 0.1, 100 ** -0.75], rtol=1e-15)
    assert np.allclose(nn.rotary_frequencies(8, 100.0, "linear", 4.0).numpy(), f / 4, rtol=1e-15)
    base = nn.rotary_frequencies(8, 100.0, "base", 4.0).numpy()
    assert base[0] == 1 and abs(base[-1] / (f[-1] / 4) - 1) < 1e-14 and (np.diff(base / f) < 0).all()
    bands = nn.rotary_frequencies(64, 10000.0, "bands", 8.0, original_tokens=4096).numpy() / nn.rotary_frequencies(64).numpy()
    turns = 4096 * nn.rotary_frequencies(64).numpy() / (2 * np.pi)
    assert (bands[turns >= 32] == 1).all() and np.allclose(bands[turns <= 1], 1 / 8) and (np.diff(bands) <= 0).all()
    assert nn.rotary_frequencies(0).numel() == 0 and nn.rotary_frequencies(2, scaling="base", factor=2.0).tolist() == [1.0]
    for bad in (dict(rotated=3), dict(rotated=8, scaling="other"), dict(rotated=8, scaling="bands"), dict(rotated=8, factor=0.0),
                dict(rotated=8, scaling="bands", original_tokens=10, slow=2.0, fast=2.0)):
        with pytest.raises(ValueError):
            nn.rotary_frequencies(**bad)


def test_layers_refuse_partitions_that_split_heads_and_positions_they_cannot_know():
    from distdl_amd.backends.stub_hip import SimWorld
    P_world = SimWorld(2).partition(0)
    P = P_world.create_partition_inclusive([0, 1])
    with pytest.raises(ValueError, match="partitioned as"):
        nn.DistributedRotary(P.create_cartesian_topology_partition([1, 1, 1, 2]), 8, device="cpu")
    with pytest.raises(ValueError, match="cannot turn"):
        nn.DistributedRotary(P.create_cartesian_topology_partition([1, 1, 2, 1]), 8, rotated=10, device="cpu")
    layer = nn.DistributedRotary(P.create_cartesian_topology_partition([1, 2, 1, 1]), 8, device="cpu")
    with pytest.raises(ValueError, match="positions"):
        layer(torch.zeros(1, 2, 1, 8))
    with pytest.raises(ValueError, match="built for"):
        layer(torch.zeros(1, 2, 1, 16))


def test_rotation_of_the_oracle_keeps_lengths_and_turns_back():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((2, 5, 3, 16))
    f, p = 10.0 ** -np.arange(6), rng.integers(0, 100, (2, 5))
    for interleaved in (False, True):
        y = o_heads.rotate(x, f, p, interleaved)
        assert np.allclose((y * y).sum(-1), (x * x).sum(-1)) and np.array_equal(y[..., 12:], x[..., 12:])
        assert np.allclose(o_heads.rotate(y, f, p, interleaved, inverse=True), x)
