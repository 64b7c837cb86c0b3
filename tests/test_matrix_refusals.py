"""Shapes the orthogonalisation refuses have no workspace, and a Muon step asks before it launches (CPU)."""

from __future__ import annotations

import pytest
from sr_states import _lib
from sr_states.hip.muon import _workspace_bytes


@pytest.mark.parametrize("rows, cols", [((1 << 20) + 1, 2), (2, (1 << 20) + 1), (1 << 20, 1 << 12), (46341, 46342)])
def test_refused_shapes_have_no_workspace(rows, cols):
    assert _lib.library().sr_orthogonalize_workspace(1, rows, cols) == 0
    with pytest.raises(ValueError, match="too large"):
        _workspace_bytes(1, rows, cols)


@pytest.mark.parametrize("rows, cols", [(1 << 20, 2), (1 << 20, 1 << 11), (46340, 46340)])
def test_the_largest_shapes_have_one(rows, cols):
    assert _workspace_bytes(3, rows, cols) >= 10 * rows * cols
