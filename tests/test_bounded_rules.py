"""A paged cache in bounded memory, without a GPU: calls whose arguments meet one another, and what the cache refuses
to give up or to reserve."""

import ctypes

import pytest
import torch

from tests.test_paged_host import block, lib  # noqa: F401


@pytest.mark.parametrize("offset", [0, 4, -4])
def test_new_lengths_over_the_old_ones_are_refused(lib, offset):
    """Blocks read the lengths while others write the new ones.  (No workspace: nothing is launched either way.)"""
    p = block(weight=4096)
    evict = lambda new: lib.rfsn_paged_evict(ctypes.byref(p), 16, 4, 4, new, None, 0, None)
    assert evict(p.lens + offset) == -1
    assert b"new_lens" in lib.rfsn_last_error(), lib.rfsn_last_error()
    for apart in (8, -8):  # two sequences' lengths further on, or before
        assert evict(p.lens + apart) == -1
        assert b"workspace" in lib.rfsn_last_error(), lib.rfsn_last_error()
