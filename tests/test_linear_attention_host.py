"""What the linear-attention layer's operators refuse, and the checked offsets: no GPU needed."""

import pytest
import torch

import pararnn_amd as P
from oracle import linear_attention as O


def test_offsets_are_checked_once():
    p = P.PackedSequences(torch.tensor([0, 3, 3, 10]))
    assert p.sequences == 3 and p.tokens == 10
    assert p.offsets(torch.device("cpu")).dtype == torch.int32
    assert p.offsets(torch.device("cpu")).tolist() == [0, 3, 3, 10]
    for bad in ([1, 3], [0, 5, 4], [0, 1 << 30]):
        with pytest.raises(ValueError):
            P.PackedSequences(torch.tensor(bad))
    for bad in (torch.zeros(1, dtype=torch.long), torch.zeros(2, 2, dtype=torch.long)):
        with pytest.raises(ValueError):
            P.PackedSequences(bad)
    with pytest.raises(TypeError):
        P.PackedSequences(torch.tensor([0.0, 2.0]))


def test_cpu_tensors_are_refused():
    q = torch.zeros(1, 4, 2, 8)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        P.linear_attention(q, q, q, torch.zeros(2))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        P.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], torch.zeros(2), torch.zeros(1, 2, 8, 8))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        P.group_norm(torch.zeros(2, 8), 2)
    used, pool = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 3)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        P.take_pages(used, 1)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        P.copy_pages(pool, torch.tensor([0]), torch.tensor([1]))


def test_oracle_packed_is_each_sequence_alone():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(1, 9, 2, 4, generator=g, dtype=torch.float64) for _ in range(3))
    a = -torch.rand(1, 9, 2, generator=g, dtype=torch.float64)
    out, state = O.linear_attention(q, k, v, a, cu=[0, 4, 4, 9])
    one, s = O.linear_attention(q[:, 4:], k[:, 4:], v[:, 4:], a[:, 4:])
    assert torch.equal(out[:, 4:], one) and torch.equal(state[2:], s)
    assert torch.equal(state[1], torch.zeros(2, 4, 4, dtype=torch.float64))


def test_c_entries_refuse_before_any_device_work():
    import ctypes
    import os

    from pararnn_amd import _lib

    if not os.path.exists(_lib.lib_path()):
        pytest.skip("library not built")
    lib = _lib.load()
    view = _lib.LaView(None, 0, 0, 0, 1)
    p = _lib.LaProblem(view, view, view, None, 0, 0, 0, None, None, None, 0, 0, 1, 8, 1, 4, 4, 0, 0,
                       1.0)
    assert lib.prnn_linear_attention_workspace_size(ctypes.byref(p)) == 0
    args = (ctypes.byref(p), ctypes.byref(view), None, None, 0, None, 0, None)
    assert lib.prnn_linear_attention(*args) == _lib.PRNN_ERR_VALUE
    assert b"non-null" in lib.prnn_last_error()
    p.dtype = 9
    assert lib.prnn_linear_attention(*args) == _lib.PRNN_ERR_TYPE
    p.dtype, p.Dk = 0, 257
    assert lib.prnn_linear_attention(*args) == _lib.PRNN_ERR_VALUE
    assert b"257" in lib.prnn_last_error()
    assert lib.prnn_group_norm(None, None, None, None, None, None, 1, 1, 8, 3, 1e-5, 0, 0, 0, None,
                               0, None) == _lib.PRNN_ERR_VALUE
    assert lib.prnn_group_norm(None, None, None, None, None, None, 1, 1, 8, 2, 1e-5, 7, 0, 0, None,
                               0, None) == _lib.PRNN_ERR_VALUE
    assert lib.prnn_pages_take(None, 4, None, 1, None) == _lib.PRNN_ERR_VALUE
    assert lib.prnn_pages_take(None, -1, None, 1, None) == _lib.PRNN_ERR_VALUE


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: without a device only")
def test_c_entries_refuse_grids_that_pass_32_bits():
    import ctypes
    import os

    from pararnn_amd import _lib

    if not os.path.exists(_lib.lib_path()):
        pytest.skip("library not built")
    lib = _lib.load()
    view = _lib.LaView(256, 8, 8, 8, 64)
    # 2^20 single tokens of 64 heads: 2^26 workgroups of 64 threads at least
    p = _lib.LaProblem(view, view, view, 256, 64, 64, 1, None, None, None, 0, 0, 1 << 20, 1, 64, 8,
                       8, 0, 0, 1.0)
    args = (ctypes.byref(p), ctypes.byref(view), None, None, 0, None, 0, None)
    assert lib.prnn_linear_attention(*args) == _lib.PRNN_ERR_VALUE
    assert b"too many for a launch" in lib.prnn_last_error()
    for n, groups in ((1 << 24, 1), (1 << 20, 64)):
        rc = lib.prnn_group_norm(256, None, None, None, 256, None, n, 2, 64, groups, 1e-5, 0, 0, 0,
                                 256, 1 << 40, None)
        assert rc == _lib.PRNN_ERR_VALUE and b"too many for a launch" in lib.prnn_last_error()
    pool = (_lib.Pool * 1)(_lib.Pool(256, 1 << 39))
    rc = lib.prnn_pages_copy(1, pool, 1, 256, 256, 1, None)
    assert rc == _lib.PRNN_ERR_VALUE and b"too many for a launch" in lib.prnn_last_error()


def test_packed_sequences_know_their_longest():
    from pararnn_amd import PackedSequences

    for cu, longest in (([0, 3, 3, 10], 7), ([0, 0], 0), ([0, 5], 5), ([0, 1, 2, 3], 1)):
        packed = PackedSequences(torch.tensor(cu))
        assert (packed.longest, packed.tokens, packed.sequences) == (longest, cu[-1], len(cu) - 1)
