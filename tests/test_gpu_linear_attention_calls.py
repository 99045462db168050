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


def _rel(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    assert got.shape == want.shape
    return float((got - want).norm() / want.norm())


def _prompts(lens, dtype, H=2, D=32, seed=1):
    n = sum(lens)
    q, k, v = (_t(1, n, H, D, dtype=dtype, seed=seed + i, scale=0.5) for i in range(3))
    g = -_t(1, n, H, dtype=dtype, seed=seed + 7).abs() / 4
    cu = [0]
    for x in lens:
        cu.append(cu[-1] + x)
    return q, k, v, g, cu


@pytest.mark.parametrize("lens", [[40, 1, 90], [700, 30, 900]], ids=["whole", "cut"])
def test_new_sessions_on_used_slots(lens):
    """A slot keeps the state of the session that had it: a new one starts from zeros all the same, alone
    and next to sessions that go on.  float32, the tests' tolerance of states."""
    from pararnn_amd import free_pages, linear_attention, take_pages

    q, k, v, g, cu = _prompts(lens, F32)
    pool = _t(6, 2, 32, 32, seed=5)
    used = torch.ones(6, dtype=torch.int32, device=DEV)
    free_pages(used, torch.tensor([4, 1, 2]))
    slots = take_pages(used, 3)
    assert slots.tolist() == [1, 2, 4]
    before = pool.clone()
    o64, s64 = O.linear_attention(*(x.double().cpu() for x in (q, k, v, g)), cu=cu)
    with torch.no_grad():
        out = linear_attention(q, k, v, g, cu_seqlens=torch.tensor(cu), block_table=slots,
                               state_out=pool)
    assert _rel(out, o64) <= 2.7e-6 and _rel(pool[slots.long()], s64) <= 2.7e-6
    assert torch.equal(pool[[0, 3, 5]], before[[0, 3, 5]])

    # the first and the last go on, the second gives its slot to a new one; in place
    now = pool.clone()
    h0 = torch.stack([now[1], torch.zeros_like(now[0]), now[4]])
    o64, s64 = O.linear_attention(*(x.double().cpu() for x in (q, k, v, g)), h0.double().cpu(), cu=cu)
    with torch.no_grad():
        out = linear_attention(q, k, v, g, h0=pool, cu_seqlens=torch.tensor(cu),
                               block_table=torch.tensor([1, -1, 4]), state_out=pool,
                               state_table=torch.tensor([1, 2, 4]))
    assert _rel(out, o64) <= 2.7e-6 and _rel(pool[[1, 2, 4]], s64) <= 2.7e-6
    assert torch.equal(pool[[0, 3, 5]], before[[0, 3, 5]])


def test_state_tables_refuse():
    from pararnn_amd import linear_attention

    q, k, v, g, _ = _prompts([8], F32)
    pool, one = _t(4, 2, 32, 32), torch.tensor([2])
    with pytest.raises(ValueError, match="state_out"):
        linear_attention(q, k, v, g, block_table=one)
    with pytest.raises(ValueError, match="block_table"):
        linear_attention(q, k, v, g, block_table=one, state_out=pool, state_table=one)
    with pytest.raises(ValueError, match="state_out"):
        linear_attention(q, k, v, g, h0=pool, block_table=one, state_table=one)
    with pytest.raises(ValueError, match="state_table"):
        linear_attention(q, k, v, g, state_out=pool, state_table=torch.tensor([1, 2]))
    with pytest.raises(ValueError, match="state_out"):
        linear_attention(q, k, v, g, state_out=pool)  # four rows for one sequence
    with pytest.raises(RuntimeError, match="inference"):
        linear_attention(q.requires_grad_(True), k, v, g, block_table=one, state_out=pool)


def test_tables_name_no_slot_beyond_32_bits():
    """Entries of 64 bits that 32 cannot hold are idle rows, not the slot that is left of them."""
    from pararnn_amd import linear_attention, linear_attention_step

    pool = _t(6, 2, 32, 32, seed=5)
    table = torch.tensor([(1 << 32) + 3, 2, -(1 << 40), 1 << 32])
    q, k, v = (_t(4, 5, 2, 32, seed=i) for i in range(3))
    g = -_t(4, 5, 2).abs()
    for call in ("prompt", "step"):
        mine = pool.clone()
        with torch.no_grad():
            if call == "prompt":
                out = linear_attention(q, k, v, g, h0=mine, block_table=table, state_out=mine)
                zeros = linear_attention(q, k, v, g)
            else:
                first = [x[:, 0] for x in (q, k, v, g)]
                out = linear_attention_step(*first, mine, block_table=table)
                zeros = linear_attention_step(*first, torch.zeros(4, 2, 32, 32, device=DEV))
        assert torch.equal(out[[0, 2, 3]], zeros[[0, 2, 3]]), call
        assert not torch.equal(mine[2], pool[2]), call
        assert torch.equal(mine[[0, 1, 3, 4, 5]], pool[[0, 1, 3, 4, 5]]), call


def test_masks_are_no_tables():
    from pararnn_amd import free_pages, linear_attention, linear_attention_step

    pool = _t(2, 2, 32, 32)
    q, g = _t(2, 3, 2, 32), -_t(2, 3, 2).abs()
    mask = torch.tensor([True, False])
    with torch.no_grad():
        with pytest.raises(TypeError, match="whole numbers"):
            linear_attention(q, q, q, g, h0=pool, block_table=mask)
        with pytest.raises(TypeError, match="whole numbers"):
            linear_attention_step(q[:, 0], q[:, 0], q[:, 0], g[:, 0], pool, block_table=mask)
    with pytest.raises(TypeError, match="whole numbers"):
        free_pages(torch.ones(2, dtype=torch.int32, device=DEV), mask)


def test_forward_mode_is_refused():
    """A dual tensor's tangent would be dropped without a word."""
    from torch.autograd import forward_ad

    from pararnn_amd import group_norm, linear_attention, linear_attention_step

    q, g, state = _t(1, 6, 2, 32), -_t(1, 6, 2).abs(), _t(1, 2, 32, 32)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(q, torch.ones_like(q))
        for call in (lambda: linear_attention(q, dual, q, g),
                     lambda: linear_attention(q, q, q, g, h0=forward_ad.make_dual(state, state)),
                     lambda: linear_attention_step(dual[:, 0], q[:, 0], q[:, 0], g[:, 0], state),
                     lambda: group_norm(dual.flatten(-2), 2),
                     lambda: group_norm(q.flatten(-2), 2, gate=dual.flatten(-2))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    call()
        assert linear_attention(q, q, q, g).shape == q.shape  # no dual among them


def test_writes_in_place_are_seen_by_autograd():
    """What saved a state that a call then overwrites refuses its backward pass; what a call would write
    in place does not require a gradient."""
    from pararnn_amd import (compact_pages, copy_pages, fork_pages, free_pages, linear_attention,
                             linear_attention_step, take_pages)

    q, g = _t(2, 6, 2, 32), -_t(2, 6, 2).abs()
    one, first = torch.tensor([0]), [q[:, 0], q[:, 0], q[:, 0], g[:, 0]]
    dest = torch.empty(2, 2, 32, device=DEV)
    used = torch.ones(2, dtype=torch.int32, device=DEV)
    used[1] = 0

    def writers(state, used):
        return {
            "prompt": lambda: linear_attention(q, q, q, g, state_out=state),
            "step": lambda: linear_attention_step(*first, state),
            "fork": lambda: fork_pages(used, state, one),
            "copy": lambda: copy_pages(state, one, one + 1),
            "compact": lambda: compact_pages(used, state)}

    for name in writers(None, None):
        leaf = q.clone().requires_grad_(True)
        state = _t(2, 2, 32, 32)
        y = linear_attention(leaf, q, q, g, h0=state).square().sum()
        with torch.no_grad():
            writers(state, used.clone())[name]()
        with pytest.raises(RuntimeError, match="inplace"):
            y.backward()
        with pytest.raises(RuntimeError, match="no_grad"):
            writers(_t(2, 2, 32, 32).requires_grad_(True), used.clone())[name]()
    table = torch.zeros(1, dtype=torch.int32, device=DEV)
    for t, call in ((dest, lambda: linear_attention_step(*first, _t(2, 2, 32, 32), out=dest)),
                    (used, lambda: take_pages(used, 1)), (used, lambda: free_pages(used, one)),
                    (table, lambda: compact_pages(used, _t(2, 3), table))):
        before = t._version
        call()
        assert t._version > before
