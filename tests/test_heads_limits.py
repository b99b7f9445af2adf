"""What the C entry points of the heads' operators say to extents that they do not take; no GPU."""

import pytest

from distdl_amd import _lib


@pytest.mark.parametrize("extents", [(1, 1, 1024, 1, 2, 64), (1, 1, 1024, 0, 2, 64), (1, 1, 1024, 3, 2, 64), (1, 1, 1024, 2, 0, 64), (1, 1, 1024, 2, -1, 64),
                                     (1 << 62, 1, 1024, 4, 4, 64), (1, 1 << 62, 1024, 4, 4, 64), (1, 1, 1 << 62, 4, 4, 64), (1, 1, 1024, 1 << 62, 1 << 62, 64),
                                     (-1, 1, 1024, 1, 1, 64), (1, 1, -1, 1, 1, 64), (1, 1, 1024, 1, 1, 0), (1, 1, 1024, 1, 1, 136)])
def test_workspaces_of_extents_that_are_refused(extents):
    """None is asked for (more key heads than heads ended the process)."""
    lib = _lib.load()
    assert lib.ddl_attention_workspace(*extents) == 0
    assert lib.ddl_attention_backward_workspace(*extents) == 0


def _attention(lib, batch, tokens, keys, heads, kv_heads, dim, dtype=_lib.DDL_DT_BF16, lse=None):
    st = _lib.i64_array((64, 128, 64))
    return lib.ddl_attention(16, st, 16, st, 16, st, dtype, batch, tokens, keys, heads, kv_heads, dim, None, 0, 0.125, 16, st, None, lse, 16, 1 << 40, None)


def _adjoint(lib, batch, tokens, keys, heads, kv_heads, dim, dtype=_lib.DDL_DT_BF16):
    st = _lib.i64_array((64, 128, 64))
    return lib.ddl_attention_backward(*[16, st] * 5, None, 16, dtype, batch, tokens, keys, heads, kv_heads, dim, None, 0, 0.125, *[16, st] * 3, 16, 1 << 40, None)


@pytest.mark.parametrize("extents", [(1 << 20, 1, 1, 16, 16, 8), (1 << 20, 1, 1, 16, 1, 8), (1 << 24, 200, 1, 1, 1, 64), (1 << 23, 129, 1, 1, 1, 64)])
def test_launches_of_2_to_32_threads_are_refused(extents):
    """256 threads for 128 queries of a head: at 2^24 workgroups no launch is possible, so none is tried."""
    lib = _lib.load()
    refusals = [lambda: _adjoint(lib, *extents), lambda: _attention(lib, *extents, lse=16)]
    if extents[4] == extents[3]:      # (few queries of heads that share a key head need fewer workgroups)
        refusals.append(lambda: _attention(lib, *extents))
    for call in refusals:
        assert call() == -5 and "2^32" in lib.ddl_last_error().decode()


@pytest.mark.parametrize("dim,dtype,sequences", [(128, _lib.DDL_DT_BF16, 1 << 23), (72, _lib.DDL_DT_F16, 1 << 23), (64, _lib.DDL_DT_F16, 1 << 24), (128, _lib.DDL_DT_F32, 1 << 24)])
def test_nothing_is_kept_for_an_adjoint_that_cannot_be_launched(dim, dtype, sequences):
    """512 threads for 128 keys of a key head in 16-bit types above 64 elements, 256 elsewhere."""
    lib = _lib.load()
    assert _attention(lib, sequences, 1, 1, 1, 1, dim, dtype, lse=16) == -5 and "2^32" in lib.ddl_last_error().decode()
    assert _adjoint(lib, sequences, 1, 1, 1, 1, dim, dtype) == -5 and "2^32" in lib.ddl_last_error().decode()
