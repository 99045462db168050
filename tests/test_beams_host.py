"""Sizes of beam selection that 32 bits cannot hold."""

import os

import pytest

from pararnn_amd import _lib

built = pytest.mark.skipif(not os.path.exists(_lib.lib_path()), reason="library not built")


@built
def test_workspaces_of_the_largest_vocabularies():
    """One beam of 2^31 - 1 tokens has slices like others: their number does not wrap."""
    size = _lib.load().prnn_beam_select_workspace_size
    for V in ((1 << 31) - 1, (1 << 31) - 8000, 1 << 30):
        per_token = size(1, 1, V, 128) / V
        assert 0.9 < per_token / (size(1, 1, 1 << 24, 128) / (1 << 24)) < 1.1
    assert size(1, 1, 1, 1) > 0
