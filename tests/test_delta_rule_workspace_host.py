"""What the delta rule asks for of memory, from its C entries: made-up addresses, none of which is used."""

import ctypes
import os

import pytest

from pararnn_amd import _lib

built = pytest.mark.skipif(not os.path.exists(_lib.lib_path()), reason="library not built")


def _problem(T, n_seq, longest, H=16, Dk=128, Dv=128, dtype=1):
    view = lambda d: _lib.LaView(4096, T * H * d, H * d, d, H)  # noqa: E731
    la = _lib.LaProblem(view(Dk), view(Dk), view(Dv), 4096, T * H, H, 1, None, None, 4096, 0, n_seq, 1, T, H, Dk,
                        Dv, dtype, dtype, 1.0, longest)
    return _lib.DeltaProblem(la, 4096, T * H, H, 1, dtype)


@built
@pytest.mark.parametrize("dtype", [0, 1], ids=["f32", "bf16"])
@pytest.mark.parametrize("short,many", [(8, 1024), (1, 4096), (100, 300)])
def test_short_sequences_take_nothing_of_a_cut_one(short, many, dtype):
    """One prompt of 16384 tokens among short ones: what its pieces take is bounded by the stream's length
    (64 pieces at most, a state and a transfer between two of them), not by the number of sequences."""
    lib = _lib.load()
    T = 16384 + short * many
    piece = 4 * 16 * 128 * 128 + 6 * 16 * 128 * 128
    for size in (lambda p: lib.prnn_delta_rule_workspace_size(ctypes.byref(p), 0),
                 lambda p: lib.prnn_delta_rule_backward_workspace_size(ctypes.byref(p), 1)):
        cut, uncut = (size(_problem(T, many + 1, longest, dtype=dtype)) for longest in (16384, 64))
        assert uncut > 0 and cut > uncut  # the long one is cut
        assert cut - uncut <= 64 * (T / 16384) * piece + (1 << 20)


@built
def test_pieces_of_rectangular_batches():
    """Between n pieces lie n - 1 states."""
    lib = _lib.load()

    def size(T):
        view = _lib.LaView(4096, T * 64, 64, 64, 1)
        la = _lib.LaProblem(view, view, view, 4096, T, 1, 1, None, None, None, 0, 0, 1, T, 1, 64, 64, 1, 1, 1.0, 0)
        return lib.prnn_delta_rule_workspace_size(ctypes.byref(_lib.DeltaProblem(la, 4096, T, 1, 1, 1)), 1)

    # (kept given: nothing but pieces' states and transfers is left)
    assert size(64) == 0
    assert size(16384) % 256 == 0 and 0 < size(16384) <= 63 * (4 * 64 * 64 + 6 * 64 * 64) + 512
