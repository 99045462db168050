"""A sample of nearly 2^31 tokens: rows are counted past the last one by a workgroup's step, which must
not wrap.  (The first version's signed count could read far outside the sample there.)"""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def test_sample_of_nearly_2_31_tokens():
    """Values and input gradients at both ends and in the middle against float64 sums: one rounding to
    float16, 2^-11, of results of the order of one."""
    from pararnn_amd import group_norm

    L, part = (1 << 31) - 1000, 1 << 27
    r = torch.Generator(device=DEV).manual_seed(3)
    x = torch.empty(1, L, 1, dtype=torch.float16, device=DEV)
    gy = torch.empty_like(x)
    for a in range(0, L, part):
        n = min(part, L - a)
        x[0, a:a + n, 0] = torch.randn(n, device=DEV, generator=r) + 0.5
        gy[0, a:a + n, 0] = torch.randn(n, device=DEV, generator=r)
    parts = [slice(a, min(a + part, L)) for a in range(0, L, part)]
    mean = sum(x[0, p].double().sum() for p in parts) / L
    var = sum((x[0, p].double() - mean).square().sum() for p in parts) / L
    rstd = 1 / torch.sqrt(var + 1e-5)
    m1 = sum(gy[0, p].double().sum() for p in parts) / L
    m2 = sum((gy[0, p].double() * (x[0, p].double() - mean) * rstd).sum() for p in parts) / L
    y = group_norm(x.requires_grad_(True), 1, over="sample")
    dx = torch.autograd.grad(y, x, gy)[0]
    for p in (slice(0, 3000), slice(L // 2, L // 2 + 3000), slice(L - 3000, L)):
        h = (x[0, p].detach().double() - mean) * rstd
        want = rstd * (gy[0, p].double() - m1 - h * m2)
        for got, e in ((y[0, p].detach(), h), (dx[0, p], want)):
            assert float((got.double() - e).norm() / e.norm()) <= 2.0 ** -11
