"""Beam selection and the pages that follow it, against sorted candidates in float64 and lists.

Parents and tokens are equal; a score is a float64 total rounded once (half a step, 2^-24 of it) after a
sum of at most 2^17 exponentials in float32 whose error, 2^-22 each at most, moves the logarithm by
2^-22: 2^-22 absolute and 2^-23 relative bound it."""

import pytest
import torch

from oracle import delta_rule as O

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")


def _check(logits, scores, beams=None, ended=None, pad=0):
    from pararnn_amd import beam_select

    want = O.beam_select(logits, scores, beams or logits.shape[1], ended, pad)
    got = beam_select(logits.to(DEV), scores.to(DEV), beams=beams,
                      ended=None if ended is None else ended.to(DEV), pad=pad)
    s, p, t = (x.cpu() for x in got)
    assert s.dtype == F32 and p.dtype == t.dtype == torch.int32
    for b, rows in enumerate(want):
        n = len(rows)
        assert p[b, :n].tolist() == [r[1] for r in rows]
        assert t[b, :n].tolist() == [r[2] for r in rows]
        for x, r in zip(s[b, :n].tolist(), rows):
            assert abs(x - r[0]) <= 2.0 ** -22 + 2.0 ** -23 * abs(r[0])
        assert (s[b, n:] == -INF).all() and (p[b, n:] == -1).all() and (t[b, n:] == -1).all()


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", [(1, 1, 1, None), (2, 3, 5, None), (1, 4, 1000, None), (3, 2, 8191, 7),
                                  (2, 8, 8193, None), (1, 1, 50257, 128), (2, 5, 20011, None),
                                  (1, 130, 33, 100), (1, 33, 9000, 64)],
                         ids=lambda c: f"B{c[0]}K{c[1]}V{c[2]}M{c[3]}")
def test_select(case, dtype):
    B, K, V, M = case
    print(f"case beams {case} {dtype}", flush=True)
    r = torch.Generator().manual_seed(V + K)
    logits = (torch.randn(B, K, V, generator=r) * 2).to(dtype)
    _check(logits, -5 - 2 * torch.rand(B, K, generator=r), M)


def test_ties_go_to_the_lowest():
    logits = torch.zeros(2, 4, 9000)
    _check(logits, torch.zeros(2, 4))  # everything equal
    logits[:, :, 8500:] = 1.0
    _check(logits, torch.zeros(2, 4), 16)
    same = torch.randn(1, 1, 3000, generator=torch.Generator().manual_seed(1)).to(BF16)
    _check(same.expand(1, 6, 3000), torch.full((1, 6), -2.5))


@pytest.mark.parametrize("order", ["rising", "falling"])
def test_sorted_logits(order):
    x = torch.linspace(-8, 8, 20000)
    x = x if order == "rising" else x.flip(0)
    _check(x.expand(1, 2, 20000).contiguous(), torch.tensor([[-1.0, -1.5]]), 64)


def test_masks_dead_beams_and_broken_rows():
    r = torch.Generator().manual_seed(8)
    logits = torch.randn(4, 3, 700, generator=r)
    scores = -torch.rand(4, 3, generator=r)
    logits[0, :, 1:] = -INF                 # one token a beam
    scores[1, 1:] = -INF                    # a search's start
    logits[2, 0, 5], logits[2, 1, 600] = float("nan"), INF
    logits[3] = -INF                        # nothing left
    _check(logits, scores)
    _check(logits, scores, 5)
    low = torch.full((1, 2, 64), torch.finfo(F32).min)
    low[0, 1, 40:] = 0.0
    _check(low, torch.zeros(1, 2), 4)


def test_ended_beams_go_on_with_one_token():
    r = torch.Generator().manual_seed(9)
    logits = torch.randn(3, 4, 9001, generator=r)
    logits[0, 1] = float("nan")             # whatever its logits
    scores = -3 * torch.rand(3, 4, generator=r)
    ended = torch.tensor([[False, True, False, False], [True] * 4, [False, False, True, True]])
    _check(logits, scores, None, ended, pad=2)


def test_strided_logits():
    r = torch.Generator().manual_seed(10)
    big = torch.randn(2, 5, 3, 3001, generator=r).to(BF16)
    from pararnn_amd import beam_select

    on, scores = big.to(DEV), torch.zeros(2, 5, device=DEV)
    view = on[:, :, -1]                     # the last position's rows, an odd number of them apart
    got, want = beam_select(view, scores), beam_select(view.contiguous(), scores)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    _check(big[:, :, -1], torch.zeros(2, 5))


@pytest.mark.parametrize("case", [(1, 1), (1, 5), (7, 8), (2, 1024), (3, 64)],
                         ids=lambda c: f"B{c[0]}K{c[1]}")
def test_reorder(case):
    from pararnn_amd import reorder_pages

    B, K = case
    r = torch.Generator().manual_seed(K)
    slots = B * K + 5
    table = torch.randperm(slots, generator=r)[:B * K].to(torch.int32).view(B, K)
    parents = torch.randint(-1, K, (B, K), generator=r, dtype=torch.int32)
    pools = [torch.randn(slots, 3, 7, generator=r), torch.randn(slots, 2, 640, generator=r).to(BF16),
             torch.randint(0, 99, (slots, 5), generator=r, dtype=torch.int8)]
    want_table, want = [], [p.clone() for p in pools]
    for b in range(B):
        new, copies = O.reorder_pages(table[b].tolist(), parents[b].tolist())
        want_table.append(new)
        for to, src in copies.items():
            for w, p in zip(want, pools):
                w[to] = p[src]
    on, mine, tab = [p.to(DEV) for p in pools], parents.to(DEV), table.to(DEV)
    got = reorder_pages(on, tab, mine)
    assert got is tab and tab.tolist() == want_table
    assert all(torch.equal(a.cpu(), w) for a, w in zip(on, want))


def test_reorder_with_idle_slots():
    from pararnn_amd import reorder_pages

    pool = torch.arange(6.0, device=DEV)[:, None].repeat(1, 4)
    table = torch.tensor([3, -1, 5, 9], dtype=torch.int32, device=DEV)
    reorder_pages(pool, table, torch.tensor([1, 1, 0, 0], device=DEV))
    # beam 1 has no state: its second child's slot is not written
    assert table.tolist() == [-1, 5, 3, 9]
    assert pool[:, 0].tolist() == [0, 1, 2, 3, 4, 5]
