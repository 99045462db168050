"""Equal beams tie wherever their rows lie: the sum of a row's exponentials must not hang on its address,
on the tokens' order in memory's 16-byte units, or on the slices next to it.

Where totals of different beams differ, they differ as float64 totals do.  A token's exponential is off by
half a unit of 2^-50 of the row's largest (a slice's is at most that), and by 2^-52 of itself; a sum is at
least one largest, so V tokens move a total by V 2^-51 at most."""

import pytest
import torch
from test_gpu_beams import BF16, DEV, F16, F32, _check

from oracle import delta_rule as O

pytestmark = pytest.mark.gpu


def _row(V, dtype, seed=0):
    r = torch.Generator().manual_seed(V + seed)
    return (torch.randn(V, generator=r) * 2.5).to(dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("V", [501, 1000, 8175, 8176, 8177, 16353, 32001, 50257])
@pytest.mark.parametrize("M", [3, 8, 40])
def test_equal_rows(V, dtype, M):
    """K copies of one row: the largest logit of every beam in their order, then the next one's."""
    logits = _row(V, dtype).expand(1, 8, V).contiguous()
    _check(logits, torch.full((1, 8), -20.3), M)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_equal_rows_at_other_addresses(dtype):
    """One row at every place in a 16-byte unit, as beams of one search and as searches of one beam."""
    from pararnn_amd import beam_select

    V, K = 20011, 16
    row = _row(V, dtype)
    step = V + 40 - V % 8 + 1
    far = torch.zeros(K * step, dtype=dtype, device=DEV)
    view = far.as_strided((1, K, V), (K * step, step, 1))
    view.copy_(row)
    scores = torch.full((1, K), -7.1, device=DEV)
    want = O.beam_select(row.expand(1, K, V), scores.cpu(), 20)[0]
    _, p, t = beam_select(view, scores, beams=20)
    assert list(zip(p[0].tolist(), t[0].tolist())) == [(k, i) for _, k, i in want]
    s, p, t = beam_select(view.transpose(0, 1), scores.t(), beams=20)
    assert (s == s[0]).all() and (t == t[0]).all() and (p == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("K", [130, 300])
def test_equal_rows_of_many_beams(dtype, K):
    logits = _row(3001, dtype).expand(1, K, 3001).contiguous()
    _check(logits, torch.zeros(1, K), 128)


@pytest.mark.parametrize("V", [4099, 50257])
def test_totals_that_lie_close(V):
    """Beams whose rows are one row's, turned, with a score per beam that shifts the totals by a few steps
    of float32: the order is that of 64 bits.  Totals that are nearer than V 2^-50 do not occur."""
    K = 8
    row = _row(V, F32, 3)
    logits = torch.stack([row.roll(17 * k) for k in range(K)])[None]
    scores = (-5.0 + torch.randperm(K, generator=torch.Generator().manual_seed(1)) * 2.0 ** -21)[None]
    _check(logits, scores, 20)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("spread", [0.0, 1.0, 30.0, 300.0])
def test_scores_are_those_of_64_bits(dtype, spread):
    """A score is its total rounded once: half a step, 2^-24 of it, and V 2^-51."""
    from pararnn_amd import beam_select

    B, K, V = 2, 3, 50257
    r = torch.Generator().manual_seed(5)
    logits = (torch.randn(B, K, V, generator=r) * spread).to(dtype)
    s, p, t = (x.cpu() for x in beam_select(logits.to(DEV), torch.zeros(B, K, device=DEV)))
    total = torch.log_softmax(logits.double(), -1)
    b = torch.arange(B)[:, None].expand(B, K)
    want = total[b, p.long(), t.long()]
    assert ((s.double() - want).abs() <= 2.0 ** -24 * want.abs() + V * 2.0 ** -51).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
def test_totals_that_are_equal_by_their_parts(dtype):
    """Equal rows whose scores differ by as much as their logits do, all in steps of a quarter: a total is
    the score and the logit, exactly, less what the rows share.  Equal ones go to the lowest beam."""
    from pararnn_amd import beam_select

    K, V, M = 12, 700, 100
    r = torch.Generator().manual_seed(11)
    row = torch.randint(-40, 40, (V,), generator=r) / 4
    scores = -torch.randint(0, 40, (K,), generator=r) / 4
    _, p, t = beam_select(row.to(dtype).expand(1, K, V).contiguous().to(DEV), scores[None].to(DEV), beams=M)
    want = sorted((-float(scores[k] + row[i]), k, -float(row[i]), i) for k in range(K) for i in range(V))[:M]
    assert list(zip(p[0].tolist(), t[0].tolist())) == [(k, i) for _, k, _, i in want]
