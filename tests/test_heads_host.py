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


def test_frequencies_take_no_gradient():
    q, f = torch.zeros(1, 2, 1, 8), torch.ones(2, dtype=torch.float64, requires_grad=True)
    for call in (lambda: nn.rotary_shard(q, None, f), lambda: nn.head_norm_rotary_shard(q, None, None, None, f)):
        with pytest.raises(ValueError, match="gradient"):
            call()


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


def _attention(lib, **change):
    st = _i64(64, 64, 64)
    a = dict(q=16, qs=st, k=16, ks=st, v=16, vs=st, dtype=_lib.DDL_DT_BF16, batch=1, tokens=1, keys=1, heads=2, kv=1, dim=64, lengths=None, causal=0,
             scale=0.125, out=16, outs=st, rest=None, lse=None, work=None, elems=0, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    return lib.ddl_attention(*a.values())


ATTENTION_REFUSALS = [
    (dict(dtype=_lib.DDL_DT_I32), -1, "dtype"), (dict(tokens=-1), -1, "negative"), (dict(dim=136), -5, "at most 128"), (dict(dim=60), -3, "16 bytes"),
    (dict(kv=0), -4, "cannot share"), (dict(heads=3, kv=2), -4, "cannot share"), (dict(scale=0.0), -1, "positive"), (dict(scale=-1.0), -1, "positive"),
    (dict(scale=float("nan")), -1, "positive"), (dict(scale=float("inf")), -1, "positive"), (dict(scale=2e38), -1, "positive"), (dict(heads=0), -4, "without heads"), (dict(q=None), -1, "null"), (dict(v=None), -1, "null"),
    (dict(outs=None), -1, "null"), (dict(k=8), -3, "aligned"), (dict(ks=_i64(64, 60, 64)), -3, "multiples"), (dict(ks=_i64(64, 1 << 22, 64)), -5, "2^22"),
    (dict(vs=_i64(64, -64, 64)), -5, "2^22"), (dict(rest=16), -1, "rest"), (dict(rest=16, lse=16, dtype=_lib.DDL_DT_F32), -1, "rest"), (dict(rest=8, lse=16), -3, "rest"),
    (dict(tokens=1 << 30), -5, "2^30"), (dict(keys=1 << 30), -5, "2^30"),
]


@pytest.mark.parametrize("change,code,what", ATTENTION_REFUSALS)
def test_attention_refuses(change, code, what):
    lib = _lib.load()
    assert _attention(lib, **change) == code
    assert what in lib.ddl_last_error().decode()


def test_attention_of_nothing_is_no_launch():
    lib = _lib.load()
    assert _attention(lib, tokens=0, q=None, out=None) == 0
    assert _attention(lib, batch=0) == 0


def test_attention_asks_for_its_workspaces():
    lib = _lib.load()
    need = lib.ddl_attention_workspace(1, 1, 65536, 2, 1, 64)
    assert need >= 2 * 2 * 64
    assert _attention(lib, keys=65536, elems=need - 1, work=16) == -1 and "workspace" in lib.ddl_last_error().decode()
    assert _attention(lib, keys=65536, elems=need, work=8) == -3
    assert lib.ddl_attention_workspace(1, 4096, 4096, 64, 8, 128) == 0
    need = lib.ddl_attention_backward_workspace(2, 5, 7, 4, 2, 64)
    assert need >= 2 * 5 * 4
    st = _i64(64, 64, 64)
    call = [16, st] * 5 + [None, 16, _lib.DDL_DT_BF16, 2, 5, 7, 4, 2, 64, None, 0, 0.125] + [16, st] * 3
    assert lib.ddl_attention_backward(*call, 16, need - 1, None) == -1 and "workspace" in lib.ddl_last_error().decode()
    assert lib.ddl_attention_backward(*call[:11], None, *call[12:], 16, need, None) == -1 and "row sums" in lib.ddl_last_error().decode()
    assert lib.ddl_attention_backward(*call[:23], None, *call[24:], 16, need, None) == -1 and "no strides" in lib.ddl_last_error().decode()
    assert lib.ddl_attention_backward(*call[:10], 8, *call[11:], 16, need, None) == -3 and "rest" in lib.ddl_last_error().decode()
    assert lib.ddl_attention_backward(*call[:10], 16, 16, _lib.DDL_DT_F32, *call[13:], 16, need, None) == -1 and "rest" in lib.ddl_last_error().decode()


def test_attention_layers_and_functions_refuse():
    from distdl_amd.backends.stub_hip import SimWorld
    q = torch.zeros(1, 1, 2, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        nn.attention_shard(q, q, q)
    P = SimWorld(2).partition(0).create_partition_inclusive([0, 1])
    for shape in ([1, 2, 1, 1], [1, 1, 1, 2]):
        with pytest.raises(ValueError, match="whole sequences"):
            nn.DistributedAttention(P.create_cartesian_topology_partition(shape))
    with pytest.raises(ValueError, match="positive"):
        nn.DistributedAttention(P.create_cartesian_topology_partition([1, 1, 2, 1]), scale=-1.0)


def test_attention_of_the_oracle_against_its_softmax():
    rng = np.random.default_rng(1)
    q, k, v = rng.standard_normal((1, 3, 2, 4)), rng.standard_normal((1, 5, 1, 4)), rng.standard_normal((1, 5, 1, 4))
    out, lse = o_heads.attention(q, k, v, [4])
    for i in range(3):
        for h in range(2):
            s = k[0, :4, 0] @ q[0, i, h] / 2
            assert np.allclose(out[0, i, h], (np.exp(s)[:, None] * v[0, :4, 0]).sum(0) / np.exp(s).sum()) and np.isclose(lse[0, i, h], np.log(np.exp(s).sum()))
    out, lse = o_heads.attention(rng.standard_normal((1, 4, 1, 4)), k[:, :2], v[:, :2], causal=True)
    assert not out[0, :2].any() and np.isinf(lse[0, :2]).all() and np.allclose(out[0, 2], v[0, 0])
