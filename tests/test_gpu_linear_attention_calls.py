"""Calls of the linear attention that a program may well make and that once went wrong."""

import pytest
import torch

from oracle import linear_attention as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def _t(*shape, dtype=F32, seed=0, scale=1.0):
    r = torch.Generator().manual_seed(seed + sum(shape))
    return (scale * torch.randn(shape, generator=r)).to(DEV, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_one_token_of_a_time_major_layout(dtype):
    """Rows of a (time, batch, heads, width) layout with one token: what lies between tokens, more
    elements than the kernels' offsets take, is between nothing."""
    from pararnn_amd import linear_attention

    B, H, D = 2100, 16, 128
    print(f"case time-major {dtype}", flush=True)
    dense = [_t(B, 1, H, D, dtype=dtype, seed=i, scale=0.3) for i in range(3)]
    g = -_t(B, 1, H, dtype=dtype).abs()

    def time_major(x):
        rest = x.shape[2:]
        n = rest.numel()
        return x.detach().clone().as_strided(x.shape, (n, B * n, *x.detach()[0, 0].stride()))

    major = [time_major(x).requires_grad_(True) for x in dense]
    assert major[0].stride(1) == B * H * D > 1 << 22
    dense = [x.requires_grad_(True) for x in dense]
    out = linear_attention(*major, time_major(g))
    want = linear_attention(*dense, g)
    assert torch.equal(out, want)
    go = _t(B, 1, H, D, dtype=dtype, seed=9)
    for x, y in zip(torch.autograd.grad(out, major, time_major(go)),
                    torch.autograd.grad(want, dense, go)):
        assert torch.equal(x, y)
