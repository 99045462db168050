"""Checked offsets handed to the recurrent cells and layers: no GPU needed."""

import pytest
import torch

from pararnn_amd import PackedSequences, ParaGRU, ParaRNN, ParaSLSTM, sequential_apply
from pararnn_amd.ragged import longest_sequence, validate_cu_seqlens


@pytest.mark.parametrize("make", [lambda: ParaSLSTM(6, 8, mix="diag"), lambda: ParaGRU(6, 8, mix="diag")],
                         ids=["slstm", "gru"])
def test_cells_take_checked_offsets(make):
    torch.manual_seed(0)
    cell, x, cu = make(), torch.randn(1, 9, 6), torch.tensor([0, 4, 5, 9])
    assert torch.equal(sequential_apply(cell, x, cu_seqlens=PackedSequences(cu)),
                       sequential_apply(cell, x, cu_seqlens=cu))


def test_layers_take_checked_offsets():
    torch.manual_seed(0)
    m = ParaRNN(ParaSLSTM(4, 8), num_layers=2).eval()
    x, cu = torch.randn(1, 9, 4), torch.tensor([0, 4, 9])
    with torch.no_grad():
        assert torch.equal(m(x, cu_seqlens=PackedSequences(cu)), m(x, cu_seqlens=cu))


def test_cells_rules_hold_for_checked_offsets():
    """As for a tensor: the last offset is the stream's length, and no sequence is empty."""
    packed = PackedSequences(torch.tensor([0, 4, 4, 9], dtype=torch.int32))
    assert packed.shortest == 0
    with pytest.raises(ValueError, match="strictly increasing"):
        validate_cu_seqlens(packed, 9)
    with pytest.raises(ValueError, match="time=8"):
        validate_cu_seqlens(PackedSequences(torch.tensor([0, 9])), 8)
    packed = PackedSequences(torch.tensor([0, 2, 9]))
    cs = validate_cu_seqlens(packed, 9)
    assert cs.dtype == torch.long and cs.tolist() == [0, 2, 9]
    assert validate_cu_seqlens(cs, 9) is cs and longest_sequence(cs, 9) == 7
    # the handle's copies are its own: a change of the given tensor is none of the batch
    given = torch.tensor([0, 2, 9])
    packed = PackedSequences(given)
    given[1] = 5
    assert validate_cu_seqlens(packed, 9).tolist() == [0, 2, 9]
    assert packed.offsets(torch.device("cpu")).tolist() == [0, 2, 9]
