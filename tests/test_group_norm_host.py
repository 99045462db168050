"""What the group norm asks for: no GPU needed."""

import os

import pytest

from pararnn_amd import _lib

pytestmark = pytest.mark.skipif(not os.path.exists(_lib.lib_path()), reason="library not built")


def test_workspace_of_aligned_arrays():
    """A group that fits a wave's registers by 16-byte accesses, and by no smaller ones, needs partial
    sums per workgroup: not per token, as arrays off the boundary would."""
    size = _lib.load().prnn_group_norm_workspace_size
    any_, aligned = (size(65536, 1, 2048, 1, _lib.PRNN_BF16, k) for k in (1, 3))
    assert any_ == 4 * 2 * 2048 * 65536 + 4 * 2 * 65536
    assert aligned <= 1024 * 2 * 2048 * 4
    for n, length, c, groups, dtype in ((5, 1, 64, 4, 0), (3, 700, 96, 8, 1), (9, 1, 5000, 1, 2),
                                        (1, 1, 1, 1, 0), (300, 7, 50, 1, 1)):
        for backward in (0, 1):
            least = size(n, length, c, groups, dtype, backward | 2)
            assert least <= size(n, length, c, groups, dtype, backward)
            token = length == 1 and c // groups <= 256 * (4 if dtype == 0 else 8)
            assert (least > 0) == (backward == 1 or not token)
