"""One handle of checked offsets for all that runs on a packed batch: the recurrent cells, a stack of
them and the linear attention."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.mark.parametrize("kind", ["slstm", "gru_head"])
def test_cells_and_linear_attention_share_a_handle(kind):
    from pararnn_amd import (NewtonConfig, PackedSequences, ParaGRU, ParaSLSTM, linear_attention,
                             newton_apply)

    torch.manual_seed(1)
    cell = {"slstm": lambda: ParaSLSTM(16, 32, mix="diag"),
            "gru_head": lambda: ParaGRU(16, 128, mix="head", n_heads=2)}[kind]().to(DEV)
    cu = torch.tensor([0, 30, 31, 190, 300])
    packed = PackedSequences(cu)
    x = torch.randn(1, 300, 16, device=DEV)
    cfg = NewtonConfig(max_iters=3, residual_atol=None, residual_fail=None)
    got = []
    for offsets in (packed, cu.to(DEV), packed):
        leaf = x.clone().requires_grad_(True)
        y = newton_apply(cell, leaf, cfg, cu_seqlens=offsets)
        got.append((y.detach(), torch.autograd.grad(y.square().sum(), leaf)[0]))
        q = x.view(1, 300, 2, 8)
        with torch.no_grad():
            linear_attention(q, q, q, torch.tensor([-0.1, -0.2], device=DEV), cu_seqlens=packed)
    for y, g in got[1:]:
        assert torch.equal(y, got[0][0]) and torch.equal(g, got[0][1])
    with pytest.raises(ValueError, match="strictly increasing"):
        newton_apply(cell, x, cfg, cu_seqlens=PackedSequences(torch.tensor([0, 30, 30, 300])))


def test_a_stack_takes_a_handle():
    from pararnn_amd import PackedSequences, ParaRNN, ParaSLSTM

    torch.manual_seed(2)
    m = ParaRNN(ParaSLSTM(16, 32), num_layers=2).to(DEV).eval()
    x, cu = torch.randn(1, 200, 16, device=DEV), torch.tensor([0, 64, 65, 200])
    with torch.no_grad():
        assert torch.equal(m(x, cu_seqlens=PackedSequences(cu)), m(x, cu_seqlens=cu))
