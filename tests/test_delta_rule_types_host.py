"""Types that the delta rule does not take are refused by name, whatever argument has them."""

import pytest
import torch

import pararnn_amd as P


@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.bool], ids=str)
@pytest.mark.parametrize("rates", [True, False], ids=["rates too", "rates in float32"])
@pytest.mark.parametrize("grads", [True, False], ids=["training", "prompt"])
def test_types_are_refused(dtype, rates, grads):
    q, g = torch.zeros(1, 4, 2, 8, dtype=dtype), torch.zeros(2).requires_grad_(grads)
    beta = torch.zeros(1, 4, 2, dtype=dtype if rates else torch.float32)
    # (on the CPU the device is what is told first)
    with pytest.raises((TypeError, RuntimeError), match="delta_rule"):
        P.delta_rule(q, q, q, g, beta)
    with pytest.raises((TypeError, RuntimeError), match="delta_rule_step"):
        P.delta_rule_step(q[:, 0], q[:, 0], q[:, 0], g.detach(), beta[:, 0], torch.zeros(1, 2, 8, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.bool], ids=str)
def test_types_are_refused_on_the_gpu(dtype):
    q = torch.zeros(1, 4, 2, 8, dtype=dtype, device="cuda:0")
    g, beta = torch.zeros(2, device="cuda:0"), torch.zeros(1, 4, 2, dtype=dtype, device="cuda:0")
    for b in (beta, beta.float()):
        with pytest.raises(TypeError, match="delta_rule supports"):
            P.delta_rule(q, q, q, g, b)
    x = torch.zeros(1, 4, 2, 8, device="cuda:0")
    with pytest.raises(TypeError, match="beta must be float32"):
        P.delta_rule(x, x, x, g, beta)
