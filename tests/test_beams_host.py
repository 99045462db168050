"""Sizes of beam selection and of the pages behind it that a launch or 32 bits cannot hold."""

import os

import pytest
import torch

from pararnn_amd import _lib

built = pytest.mark.skipif(not os.path.exists(_lib.lib_path()), reason="library not built")
no_device = pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: without a device only")


@built
def test_workspaces_of_the_largest_vocabularies():
    """One beam of 2^31 - 1 tokens has slices like others: their number does not wrap."""
    size = _lib.load().prnn_beam_select_workspace_size
    for V in ((1 << 31) - 1, (1 << 31) - 8000, 1 << 30):
        per_token = size(1, 1, V, 128) / V
        assert 0.9 < per_token / (size(1, 1, 1 << 24, 128) / (1 << 24)) < 1.1
    assert size(1, 1, 1, 1) > 0


@built
@no_device
def test_reorder_refuses_more_searches_than_a_launch_takes():
    lib = _lib.load()
    pools = (_lib.Pool * 1)(_lib.Pool(4096, 64))
    call = lambda B, K: lib.prnn_pages_reorder(4, pools, 1, 4096, 4096, B, K, 4096, None)  # noqa: E731
    for B, K in ((1 << 22, 1), (1 << 29, 2), (1 << 30, 1)):
        assert call(B, K) == _lib.PRNN_ERR_VALUE
        assert b"too many for a launch" in lib.prnn_last_error()
    assert call((1 << 22) - 1, 1) == _lib.PRNN_ERR_RUNTIME  # what fails then is the missing device
