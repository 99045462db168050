"""The example of the delta-rule block: it runs, its search's totals are those of one pass, and its
gradients are those of the same model on the operators' definitions in float64."""

import importlib.util
import os

import pytest
import torch
from conftest import REPO

from oracle import delta_rule as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _example():
    path = os.path.join(REPO, "examples", "delta_rule.py")
    spec = importlib.util.spec_from_file_location("delta_rule_example", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    return example


def test_it_trains_and_searches():
    """float32: a total is a sum of nine logarithms of at most some units, each off by the logits' own
    error (a few thousand roundings of 2^-24 in a random walk through two blocks, 1e-5)."""
    losses, off = _example().main(steps=20)
    assert len(losses) == 20 and all(x == x and x < 1e3 for x in losses)
    assert off <= 9 * 2e-5


def test_gradients(monkeypatch):
    """Every parameter's gradient of one packed batch, float32 on the GPU against float64 on the CPU:
    two blocks of five operators, each a random walk of some 2^-24 sqrt(2000) = 2.7e-6 (as the rule
    alone), forwards and backwards: sqrt(2 x 2 x 5) 2.7e-6 = 1.2e-5, and 4 for the norms' and gates'
    slopes: 5e-5."""
    example = _example()
    torch.manual_seed(3)
    model = example.Model(16, width=32, blocks=2, heads=2, d_key=16, d_value=8)
    lens = [70, 1, 29]
    cu = [0, 70, 71, 100]
    ids, _ = example.recall(16, lens, torch.Generator().manual_seed(5))
    want_ids = ids.roll(-1)

    def loss(m, ids, want, packed):
        return torch.nn.functional.cross_entropy(m(ids[None], packed)[0], want)

    mine = example.Model(16, width=32, blocks=2, heads=2, d_key=16, d_value=8).to(DEV)
    mine.load_state_dict(model.state_dict())
    got = torch.autograd.grad(
        loss(mine, ids.to(DEV), want_ids.to(DEV), example.PackedSequences(torch.tensor(cu))),
        list(mine.parameters()))
    torch.cuda.synchronize()

    def rule(q, k, v, g, b, cu_seqlens):
        return O.delta_rule(q, k, v, g, b, cu=cu_seqlens)[0]

    def group_norm(x, groups, weight, gate, activation):
        x = x.unflatten(-1, (groups, -1))
        d = x - x.mean(-1, keepdim=True)
        z = d / torch.sqrt((d * d).mean(-1, keepdim=True) + 1e-5)
        return z.flatten(-2) * weight * torch.nn.functional.silu(gate)

    monkeypatch.setattr(example, "delta_rule", rule)
    monkeypatch.setattr(example, "residual_norm", O.residual_norm)
    monkeypatch.setattr(example, "group_norm", group_norm)
    exact = model.double()
    want = torch.autograd.grad(loss(exact, ids, want_ids, cu), list(exact.parameters()))
    for (name, _), x, y in zip(exact.named_parameters(), got, want):
        off = float((x.double().cpu() - y).norm() / y.norm().clamp(min=1e-9))
        print(f"  {name} {off:.1e}", flush=True)
        assert off <= 5e-5, name
