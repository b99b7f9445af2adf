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
