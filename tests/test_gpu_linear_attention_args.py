"""Refusals of the linear-attention layer's operators on GPU tensors: each before any launch."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def _t(*shape, dtype=torch.float32):
    return torch.zeros(*shape, dtype=dtype, device=DEV)


@pytest.mark.parametrize("change,error", [
    (dict(q=lambda: _t(1, 6, 2)), ValueError),
    (dict(k=lambda: _t(1, 5, 2, 8)), ValueError),
    (dict(k=lambda: _t(1, 6, 2, 9)), ValueError),
    (dict(k=lambda: _t(1, 6, 3, 8)), ValueError),
    (dict(v=lambda: _t(1, 6, 2, 300)), ValueError),
    (dict(v=lambda: _t(1, 6, 2, 8, dtype=torch.bfloat16)), TypeError),
    (dict(q=lambda: _t(1, 6, 2, 8, dtype=torch.float64)), TypeError),
    (dict(g=lambda: _t(1, 6, 2, dtype=torch.bfloat16)), TypeError),
    (dict(g=lambda: _t(1, 7, 2)), ValueError),
    (dict(g=lambda: _t(3)), ValueError),
    (dict(g=lambda: torch.zeros(2)), RuntimeError),
    (dict(h0=lambda: _t(2, 2, 8, 8)), ValueError),
    (dict(h0=lambda: _t(1, 2, 8, 8, dtype=torch.bfloat16)), TypeError),
    (dict(cu_seqlens=lambda: torch.tensor([0, 5])), ValueError),
    (dict(cu_seqlens=lambda: torch.tensor([0, 4, 3, 6])), ValueError),
    (dict(block_table=lambda: torch.tensor([0])), ValueError),
    (dict(h0=lambda: _t(4, 2, 8, 8), block_table=lambda: torch.tensor([0, 1])), ValueError),
    (dict(h0=lambda: _t(4, 2, 8, 8), block_table=lambda: torch.tensor([0.0])), TypeError),
    (dict(state_out=lambda: _t(1, 2, 8, 9)), ValueError),
    (dict(state_out=lambda: _t(1, 2, 8, 16)[..., ::2]), ValueError),
])
def test_linear_attention_refuses(change, error):
    from pararnn_amd import linear_attention

    args = dict(q=_t(1, 6, 2, 8), k=_t(1, 6, 2, 8), v=_t(1, 6, 2, 8), g=_t(1, 6, 2))
    args.update({n: f() for n, f in change.items()})
    first = [args.pop(n) for n in "qkvg"]
    with pytest.raises(error):
        linear_attention(*first, **args)


def test_linear_attention_refuses_gradients_where_there_are_none():
    from pararnn_amd import linear_attention, linear_attention_step

    q = _t(1, 6, 2, 8).requires_grad_(True)
    with pytest.raises(RuntimeError, match="inference"):
        linear_attention(q, q, q, _t(2), h0=_t(3, 2, 8, 8), block_table=torch.tensor([1]))
    with pytest.raises(RuntimeError, match="autograd"):
        linear_attention_step(q[:, 0], q[:, 0], q[:, 0], _t(2), _t(1, 2, 8, 8))


@pytest.mark.parametrize("change,error", [
    (dict(q=lambda: _t(2, 2, 2, 8)), ValueError),
    (dict(k=lambda: _t(3, 2, 8)), ValueError),
    (dict(v=lambda: _t(2, 3, 8)), ValueError),
    (dict(g=lambda: _t(2, 3)), ValueError),
    (dict(g=lambda: _t(3, 2)), ValueError),
    (dict(state=lambda: _t(1, 2, 8, 8)), ValueError),
    (dict(state=lambda: _t(2, 2, 8, 8, dtype=torch.bfloat16)), TypeError),
    (dict(state=lambda: _t(2, 2, 8, 16)[..., ::2]), ValueError),
    (dict(block_table=lambda: torch.tensor([0, 1, 2])), ValueError),
    (dict(out=lambda: _t(2, 2, 9)), ValueError),
    (dict(out=lambda: _t(2, 2, 8, dtype=torch.bfloat16)), ValueError),
])
def test_step_refuses(change, error):
    from pararnn_amd import linear_attention_step

    args = dict(q=_t(2, 2, 8), k=_t(2, 2, 8), v=_t(2, 2, 8), g=_t(2, 2), state=_t(2, 2, 8, 8))
    args.update({n: f() for n, f in change.items()})
    first = [args.pop(n) for n in ("q", "k", "v", "g", "state")]
    with pytest.raises(error):
        linear_attention_step(*first, **args)


@pytest.mark.parametrize("kw,error", [
    (dict(num_groups=3), ValueError), (dict(num_groups=0), ValueError),
    (dict(weight=lambda: _t(7)), ValueError),
    (dict(weight=lambda: _t(8, dtype=torch.bfloat16)), TypeError),
    (dict(weight=lambda: torch.zeros(8)), RuntimeError),
    (dict(gate=lambda: _t(4, 7)), ValueError),
    (dict(gate=lambda: _t(4, 8, dtype=torch.bfloat16)), TypeError),
    (dict(activation="relu"), ValueError), (dict(over="time"), ValueError),
    (dict(eps=-1.0), ValueError),
])
def test_group_norm_refuses(kw, error):
    from pararnn_amd import group_norm

    kw = {n: f() if callable(f) else f for n, f in kw.items()}
    with pytest.raises(error):
        group_norm(_t(4, 8), kw.pop("num_groups", 2), **kw)


def test_pages_refuse():
    from pararnn_amd import compact_pages, copy_pages, fork_pages, free_pages, take_pages

    used, pool = _t(4, dtype=torch.int32), _t(4, 3)
    with pytest.raises(TypeError):
        take_pages(_t(4), 1)
    with pytest.raises(ValueError):
        take_pages(used, -1)
    with pytest.raises(ValueError):
        take_pages(_t(8, dtype=torch.int32)[::2], 1)
    with pytest.raises(ValueError):
        fork_pages(used, [pool, _t(5, 3)], torch.tensor([0]))
    with pytest.raises(TypeError):
        fork_pages(used, pool, torch.tensor([0.0]))
    with pytest.raises(ValueError):
        fork_pages(used, _t(4, 6)[:, ::2], torch.tensor([0]))
    with pytest.raises(ValueError):
        free_pages(used, torch.tensor([[0]]))
    with pytest.raises(ValueError):
        copy_pages(pool, torch.tensor([0]), torch.tensor([1, 2]))
    with pytest.raises(ValueError):
        copy_pages([], torch.tensor([0]), torch.tensor([1]))
    with pytest.raises(TypeError):
        compact_pages(used, pool, [_t(3, dtype=torch.int64)])
    with pytest.raises(ValueError):
        compact_pages(used, pool, [_t(6, dtype=torch.int32)[::2]])
    with pytest.raises(RuntimeError):
        compact_pages(used, pool, [torch.zeros(3, dtype=torch.int32)])


def test_packed_offsets_outlast_work_on_another_stream():
    """A handle dropped while a side stream has yet to read its offsets: their memory is not handed
    out before (what would lie there, all sequences empty, is valid too)."""
    from pararnn_amd import PackedSequences, linear_attention

    g = torch.Generator().manual_seed(5)
    n = 4096
    q = torch.randn(1, n, 2, 16, generator=g).to(DEV)
    a = -torch.rand(1, n, 2, generator=g).to(DEV)
    cu = torch.arange(0, n + 1, 16)
    with torch.no_grad():
        want, state = linear_attention(q, q, q, a, cu_seqlens=cu, return_state=True)
        side = torch.cuda.Stream()
        packed = PackedSequences(cu)
        linear_attention(q, q, q, a, cu_seqlens=packed)  # the copy belongs to this stream
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            got, late = linear_attention(q, q, q, a, cu_seqlens=packed, return_state=True)
        del packed
        others = [torch.zeros(cu.numel(), dtype=torch.int32, device=DEV) for _ in range(64)]
        torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(late, state) and len(others) == 64


def test_gradients_are_differentiable_once():
    """A graph of the gradients can be asked for; a second derivative is refused, not wrong."""
    from pararnn_amd import group_norm, linear_attention

    g = torch.Generator().manual_seed(9)
    q = torch.randn(1, 20, 2, 8, generator=g).to(DEV).requires_grad_(True)
    a = -torch.rand(1, 20, 2, generator=g).to(DEV)
    for y in (linear_attention(q, q, q, a), group_norm(q.flatten(-2), 2)):
        plain = torch.autograd.grad(y.square().sum(), q, retain_graph=True)[0]
        again = torch.autograd.grad(y.square().sum(), q, create_graph=True)[0]
        assert torch.equal(plain, again)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            again.sum().backward()
