"""Gradients that are not finite: by the definition one of a token's output reaches what its sequence's
earlier tokens and itself do, never a later token, another head, another sequence."""

import pytest
import torch
from test_gpu_delta_rule import BF16, F16, F32, _inputs
from test_gpu_delta_rule_calls import _on, _train

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
NAMES = ("out", "state", "dq", "dk", "dv", "dg", "dbeta", "dh0")


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("dims", [(32, 32), (64, 48), (128, 72), (256, 40)], ids=lambda d: f"D{d[0]}x{d[1]}")
def test_a_gradient_that_is_not_finite(dims, bad, dtype):
    from pararnn_amd import PackedSequences

    cu, H, (Dk, Dv), col = [0, 50, 950], 2, dims, 3
    print(f"case gradient not finite {dims} {bad} {dtype}", flush=True)
    *given, go, gs = _on(_inputs(1, cu[-1], (H, H, H), Dk, Dv, dtype, "token", 4, seqs=2))
    packed = PackedSequences(torch.tensor(cu))
    want = dict(zip(NAMES, _train(given, go, gs, cu_seqlens=packed)))
    others = [c for c in range(Dv) if c != col]
    for at in (50, 370, 500, 949):  # a sequence's first token, some in a chunk, its last
        broken = go.clone()
        broken[0, at, 1, col] = bad
        got = dict(zip(NAMES, _train(given, broken, gs, cu_seqlens=packed)))
        for name in NAMES:
            x, y = got[name], want[name]
            if name in ("out", "state"):
                assert torch.equal(x, y), name
            elif name == "dh0":
                assert torch.equal(x[0], y[0]) and torch.equal(x[:, 0], y[:, 0])
                assert torch.equal(x[..., others], y[..., others])
                assert not torch.isfinite(x[1, 1, :, col]).any()
            else:
                assert torch.equal(x[:, :, 0], y[:, :, 0]), name
                assert torch.equal(x[:, :50], y[:, :50]) and torch.equal(x[:, at + 1:], y[:, at + 1:]), (name, at)
                if name == "dq":
                    assert torch.equal(x[:, :at], y[:, :at]) and not torch.isfinite(x[0, at, 1]).any()
                elif name == "dv":
                    assert torch.equal(x[..., others], y[..., others])
                    assert not torch.isfinite(x[0, 50:at + 1, 1, col]).any()
                else:
                    assert not torch.isfinite(x[0, 50:at + 1, 1]).any(), (name, at)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("which", ["q", "k", "g", "beta"])
def test_inputs_that_are_not_finite(which, dtype):
    """A token's q, key, decay or rate: values before it have no gradient that could be finite, values
    behind its chunk have theirs, and nothing that is finite is another one's."""
    T, H, D, at = 300, 2, 64, 150
    *given, go, gs = _on(_inputs(1, T, (H, H, H), D, D, dtype, "token", 4))
    want = dict(zip(NAMES, _train(given, go, gs)))
    i = ("q", "k", None, "g", "beta").index(which)
    given[i] = given[i].clone()
    if given[i].dim() == 4:
        given[i][0, at, 1, 3] = NAN
    else:
        given[i][0, at, 1] = NAN
    got = dict(zip(NAMES, _train(given, go, gs)))
    for name in NAMES[2:]:
        assert torch.equal(got[name][:, :, 0] if name != "dh0" else got[name][:, 0],
                           want[name][:, :, 0] if name != "dh0" else want[name][:, 0]), name
    x, y = got["dv"][0, :, 1], want["dv"][0, :, 1]
    assert not torch.isfinite(x[:at]).any()
    assert torch.equal(x[192:], y[192:])
    assert ((x == y) | x.isnan()).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("bad", [NAN, INF])
def test_a_value_that_is_not_finite(bad, dtype):
    """One in v: earlier tokens' gradients are those without it, and every value's own."""
    T, H, D, at, col = 300, 2, 64, 150, 3
    *given, go, gs = _on(_inputs(1, T, (H, H, H), D, D, dtype, "token", 4))
    go[:, at:, 1, col] = 0
    gs[:, 1, :, col] = 0
    want = dict(zip(NAMES, _train(given, go, gs)))
    given[2] = given[2].clone()
    given[2][0, at, 1, col] = bad
    got = dict(zip(NAMES, _train(given, go, gs)))
    assert torch.equal(got["dv"], want["dv"]) and torch.equal(got["dh0"], want["dh0"])
    for name in ("dq", "dk", "dg", "dbeta"):
        assert torch.equal(got[name][:, :, 0], want[name][:, :, 0]), name
    assert torch.equal(got["dq"][:, :at], want["dq"][:, :at])
    assert not torch.isfinite(got["dq"][0, at:, 1]).any()
