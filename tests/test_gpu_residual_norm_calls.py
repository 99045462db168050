"""How the residual norm is called: refusals, streams, graphs, large arrays, values that are not finite,
differences.  A token's results depend on its own row alone, so equal rows are equal bits."""

import pytest
import torch
from test_gpu_residual_norm import BF16, CASES, DEV, F16, F32, _case, _rel

from oracle import delta_rule as O

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def _run(given, fixed, seeds):
    """(h, z, gradients in the order of `given`)."""
    from pararnn_amd import residual_norm

    leaves = {n: t.detach().requires_grad_(True) for n, t in given.items()}
    h, z = residual_norm(leaves["x"], leaves.get("y"),
                         **{n: t for n, t in leaves.items() if n not in ("x", "y")}, **fixed)
    return (h.detach(), z.detach(), *torch.autograd.grad([h, z], list(leaves.values()), seeds))


def _on(case, dtype, seed=0):
    given, fixed, seeds = _case(case, dtype, seed)
    return {n: t.to(DEV) for n, t in given.items()}, fixed, [t.to(DEV) for t in seeds]


def _same(a, b):
    for i, (x, y) in enumerate(zip(a, b)):
        assert torch.equal(x, y), i


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", [CASES[4], CASES[6], CASES[7]], ids=["1024", "40", "4104"])
def test_layouts_streams_and_bits(case, dtype):
    """Strided rows, parameters and arrays off a 16-byte boundary, expanded gradients, another stream."""
    print(f"case layouts {case[0]} {dtype}", flush=True)
    given, fixed, seeds = _on(case, dtype)
    want = _run(given, fixed, seeds)
    _same(_run(given, fixed, seeds), want)
    odd = lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape)  # noqa: E731
    wide = lambda t: torch.cat([t, t], -1)[..., :t.shape[-1]]  # noqa: E731
    for change in (odd, wide):
        got = _run({n: change(t) for n, t in given.items()}, fixed, [change(t) for t in seeds])
        _same(got, want)
    one = torch.ones(1, dtype=dtype, device=DEV)
    _same(_run(given, fixed, [one.expand(given["x"].shape)] * 2),
          _run(given, fixed, [one.expand(given["x"].shape).contiguous()] * 2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run({n: t * 1 for n, t in given.items()}, fixed, [t * 1 for t in seeds])
    side.synchronize()
    _same(got, want)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_captured_training(dtype):
    case = ((700, 1000), "layer", True, True, "silu", True, "vector", True, True, False)
    given, fixed, seeds = _on(case, dtype)
    leaves = {n: t.requires_grad_(True) for n, t in given.items()}

    def run():
        from pararnn_amd import residual_norm

        h, z = residual_norm(leaves["x"], leaves["y"],
                             **{n: t for n, t in leaves.items() if n not in ("x", "y")}, **fixed)
        return (h, z, *torch.autograd.grad([h, z], list(leaves.values()), seeds))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        result = run()
    for seed in (1, 2, 3):
        fresh, _, others = _on(case, dtype, seed)
        with torch.no_grad():
            for n in fresh:
                leaves[n].copy_(fresh[n])
            for t, x in zip(seeds, others):
                t.copy_(x)
        graph.replay()
        got = [t.detach().clone() for t in result]
        want = _run(fresh, fixed, others)
        torch.cuda.synchronize()
        _same(got, want)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("bad", [NAN, INF, -INF])
def test_rows_keep_to_themselves(bad, dtype):
    for width in (64, 1000, 9000):
        case = ((7, width), "layer", True, True, "silu", True, "vector", True, True, False)
        given, fixed, seeds = _on(case, dtype)
        want = _run(given, fixed, seeds)
        rows = [0, 1, 2, 4, 5, 6]
        names = list(given)
        for name in ("x", "y", "gate"):
            broken = {n: t.clone() for n, t in given.items()}
            broken[name][3, 5] = bad
            got = _run(broken, fixed, seeds)
            for i in (0, 1, *(2 + names.index(n) for n in ("x", "y", "gate"))):
                assert torch.equal(got[i][rows], want[i][rows]), (name, i)
            if name != "gate" or bad != -INF:
                assert not torch.isfinite(got[1][3]).any(), name


@pytest.mark.parametrize("width", [40, 1000, 4104, 8192, 9000])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_some_gradients_only(dtype, width):
    """A leaf alone has the gradient that it has among all."""
    from pararnn_amd import residual_norm

    case = ((9, width), "layer", True, True, "silu", True, "vector", True, True, False)
    given, fixed, seeds = _on(case, dtype)
    want = dict(zip(given, _run(given, fixed, seeds)[2:]))
    for name in given:
        leaves = dict(given)
        leaves[name] = leaves[name].detach().requires_grad_(True)
        h, z = residual_norm(**leaves, **fixed)
        out = [t for t in (h, z) if t.requires_grad]
        got, = torch.autograd.grad(out, [leaves[name]], seeds[-len(out):])
        assert torch.equal(got, want[name]), name


def test_rows_of_zeros_and_large_values():
    """A row of zeros under eps = 1e-6 and zero variance; values whose squares pass float32's range are
    the caller's, those of 1e15 are not."""
    from pararnn_amd import residual_norm

    x = torch.zeros(3, 200, dtype=torch.float32)
    x[1] = 7.0
    x[2] = torch.randn(200, generator=torch.Generator().manual_seed(1)) * 1e15
    y = torch.zeros_like(x)
    for norm in ("rms", "layer"):
        h, z = residual_norm(x.to(DEV), y.to(DEV), post_norm=True, norm=norm)
        h64, z64 = O.residual_norm(x.double(), y.double(), post_norm=True, norm=norm)
        assert torch.equal(h.cpu(), x)
        assert (z[0] == 0).all() and _rel(z[2], z64[2]) <= 2e-6
        # a constant row's mean is off by half a step of 7 at most, over sqrt(eps)
        assert float((z[1].double().cpu() - z64[1]).abs().max()) <= (7 * 2.0 ** -24 / 1e-3 if norm == "layer" else 2e-6)


@pytest.mark.parametrize("which", ["x", "y", "weight", "bias", "post_weight", "gate", "scale"])
def test_gradients_against_differences(which):
    """Along the gradient's own direction, five points in float32: the loss is off by 2e-6 of the
    results' and seeds' norms, 1.5 of that in the quotient, over a step of 0.1; sixteen rows of 24, whose
    curvature over a step of 0.1 / sqrt(24) leaves less than 1e-4 to the fourth power's term."""
    from pararnn_amd import residual_norm

    case = ((16, 24), "layer", True, True, "silu", True, "vector", True, True, False)
    given, fixed, seeds = _on(case, F32)
    h, z, *grads = _run(given, fixed, seeds)
    grad = grads[list(given).index(which)].double()
    size = float(grad.norm())
    along = (grad / size).float()

    def loss(step):
        moved = dict(given)
        moved[which] = moved[which] + step * along
        with torch.no_grad():
            out = residual_norm(**moved, **fixed)
        return sum(float((o.double() * s.double()).sum()) for o, s in zip(out, seeds))

    d = 0.1
    slope = (8 * (loss(d) - loss(-d)) - (loss(2 * d) - loss(-2 * d))) / (12 * d)
    noise = 2e-6 * 1.5 / d * sum(float(o.norm() * s.norm()) for o, s in zip((h, z), seeds))
    print(f"case differences {which}: {slope:.6f} {size:.6f} +- {noise:.1e}", flush=True)
    assert noise < 0.05 * size and abs(slope - size) <= noise + 1e-4 * size


def test_more_than_2_to_31_values():
    """131075 rows of 16384: the last rows as a call on them alone, forwards and backwards."""
    from pararnn_amd import residual_norm

    N, C, last = 131075, 16384, 5
    print("case more than 2^31 values", flush=True)
    x = torch.empty(N, C, dtype=BF16, device=DEV).normal_()
    y = torch.empty(N, C, dtype=BF16, device=DEV).normal_()
    w = torch.randn(C, device=DEV)
    gate = x.flip(0)
    ends = {}
    for name, rows in (("all", slice(None)), ("last", slice(N - last, None))):
        leaves = [t[rows].detach().requires_grad_(True) for t in (x, y, gate)]
        h, z = residual_norm(leaves[0], leaves[1], w, post_norm=True, gate=leaves[2], activation="silu")
        grads = torch.autograd.grad([h, z], leaves, [y[rows], x[rows]])
        ends[name] = [t[-last:].detach().clone() for t in (h, z, *grads)]
    _same(ends["all"], ends["last"])


def _t(*shape, dtype=F32):
    return torch.zeros(*shape, dtype=dtype, device=DEV)


@pytest.mark.parametrize("change,error", [
    (dict(x=lambda: _t(1)[0]), ValueError),
    (dict(x=lambda: _t(4, 0), y=lambda: _t(4, 0)), ValueError),
    (dict(x=lambda: _t(1, 16385), y=lambda: _t(1, 16385)), ValueError),
    (dict(x=lambda: _t(4, 8, dtype=torch.float64)), TypeError),
    (dict(x=lambda: torch.zeros(4, 8), y=lambda: torch.zeros(4, 8)), RuntimeError),
    (dict(y=lambda: _t(4, 7)), ValueError),
    (dict(y=lambda: _t(8)), ValueError),
    (dict(y=lambda: _t(4, 8, dtype=BF16)), TypeError),
    (dict(y=lambda: torch.zeros(4, 8)), RuntimeError),
    (dict(gate=lambda: _t(4, 7)), ValueError),
    (dict(gate=lambda: _t(4, 8, dtype=BF16)), TypeError),
    (dict(weight=lambda: _t(7)), ValueError),
    (dict(weight=lambda: _t(8, dtype=BF16)), TypeError),
    (dict(weight=lambda: torch.zeros(8)), RuntimeError),
    (dict(x=lambda: _t(4, 8, dtype=BF16), y=lambda: _t(4, 8, dtype=BF16), weight=lambda: _t(8),
          bias=lambda: _t(8, dtype=BF16)), TypeError),
    (dict(scale=lambda: _t(1)[0]), ValueError),
    (dict(post_weight=lambda: _t(8)), ValueError),
    (dict(activation=lambda: "silu"), ValueError),
    (dict(activation=lambda: "relu", gate=lambda: _t(4, 8)), ValueError),
    (dict(norm=lambda: "batch"), ValueError),
    (dict(eps=lambda: -1.0), ValueError),
    (dict(eps=lambda: NAN), ValueError),
    (dict(y=lambda: None, gate=lambda: _t(4, 8)), ValueError),
    (dict(y=lambda: None, scale=lambda: 0.5), ValueError),
    (dict(y=lambda: None, post_norm=lambda: True), ValueError),
])
def test_refuses(change, error):
    from pararnn_amd import residual_norm

    args = dict(x=_t(4, 8), y=_t(4, 8))
    args.update({n: f() for n, f in change.items()})
    with pytest.raises(error, match="residual_norm"):
        residual_norm(args.pop("x"), args.pop("y"), **args)


def test_autograd_once_and_no_duals():
    from torch.autograd import forward_ad

    from pararnn_amd import residual_norm

    x = torch.randn(4, 8, device=DEV).requires_grad_(True)
    h, z = residual_norm(x, x)  # one tensor twice: both gradients
    exact = x.detach().double().cpu().requires_grad_(True)
    h64, z64 = O.residual_norm(exact, exact)
    want, = torch.autograd.grad(h64.sum() + z64.square().sum(), exact)
    got, = torch.autograd.grad(h.sum() + z.square().sum(), x)
    assert _rel(got, want) <= 2e-6
    h, z = residual_norm(x, x)
    grad, = torch.autograd.grad(z.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once"):
        grad.sum().backward()
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.detach(), torch.ones(4, 8, device=DEV))
        for call in (lambda: residual_norm(dual, x), lambda: residual_norm(x, dual),
                     lambda: residual_norm(x, x, gate=dual), lambda: residual_norm(x, x, dual[0])):
            for on in (True, False):
                with torch.set_grad_enabled(on), pytest.raises(RuntimeError, match="forward-mode"):
                    call()


def test_too_many_rows():
    from pararnn_amd import residual_norm

    x = torch.zeros(1, 1, dtype=BF16, device=DEV).expand((1 << 31) + 5, 1)
    with pytest.raises(ValueError, match="2\\^31"):
        residual_norm(x, x)
