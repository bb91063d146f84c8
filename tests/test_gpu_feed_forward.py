"""The gated feed-forward block against its float64 statement (``oracle.node_ops.gated_feed_forward``, which also bounds
what the roundings of a float32 evaluation with 16-bit operands may come to, element by element)."""

import math

import pytest
import torch

from oracle import node_ops as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["silu", "sigmoid", "gelu"]
NAMES = ("y", "dx", "dw_in", "dw_out")


def _F():
    from flashcart_amd.nn import functional as F
    return F


def _inputs(n, width, hidden, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    t = [torch.randn(*s, device=DEV, generator=gen).to(dtype)
         for s in ((n, width), (2 * hidden, width), (width, hidden), (n, width))]
    return t[:3], t[3]


def _run(x, w_in, w_out, act, c, s_in, s_out, grad):
    leaves = [t.detach().requires_grad_(True) for t in (x, w_in, w_out)]
    y = _F().gated_feed_forward(*leaves, act, c, s_in, s_out)
    return dict(zip(NAMES, (y.detach(), *torch.autograd.grad(y, leaves, grad))))


def _roundings(dtype):
    u = torch.finfo(dtype).eps / 2
    if dtype == torch.float32:
        return dict(mid=0.0, end=u, kept=0.0, tiny=2.0 ** -140)
    # the kept factors hold 16 significant bits
    return dict(mid=u, end=u, kept=2.0 ** -17, tiny=2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)


def _check(got, want, dtype):
    # two independent roundings of relative size u, uniform in their interval (u / sqrt 3 each), and the kept factors;
    # float32: sums in the matrix instructions
    norm = 1e-6 if dtype == torch.float32 else 0.9 * torch.finfo(dtype).eps / 2
    for name, value in got.items():
        ref, bound = want[name]
        off = (value.double() - ref).abs()
        assert value.dtype == dtype and value.shape == ref.shape, name
        assert bool((off <= bound).all()), f"{name}: {float((off / bound).max())} times the bound"
        if ref.numel() >= 1000:
            rel = float(off.norm() / ref.norm())
            assert rel <= norm, f"{name}: relative error {rel}"


# one row, sizes of one, odd ones, more than one tile each way, long sums of few outputs (n large, width and hidden
# small; hidden large, n small), the largest tiles with and without ragged edges
SIZES = [(1, 1, 1), (1, 64, 64), (3, 5, 7), (17, 33, 19), (64, 128, 512), (130, 96, 200), (257, 519, 103),
         (1000, 64, 72), (300, 256, 1032), (5, 2056, 40), (70, 40, 3001), (9001, 24, 16), (2049, 136, 264),
         (4096, 512, 1024), (4100, 520, 1100), (16, 1024, 2048), (48, 2048, 1000), (33, 72, 4099),
         (8200, 520, 1032)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,width,hidden", SIZES)
def test_feed_forward(n, width, hidden, dtype):
    act = ACTS[(n + width + hidden) % 3]
    print(f"feed-forward n={n} width={width} hidden={hidden} {act} {dtype}", flush=True)
    (x, w_in, w_out), grad = _inputs(n, width, hidden, dtype)
    args = (act, 1.6, width ** -0.5, hidden ** -0.5)
    want = O.gated_feed_forward(x, w_in, w_out, *args, grad, **_roundings(dtype))
    got = _run(x, w_in, w_out, *args, grad)
    _check(got, want, dtype)
    with torch.no_grad():
        _check({"y": _F().gated_feed_forward(x, w_in, w_out, *args)}, want, dtype)
    again = _run(x, w_in, w_out, *args, grad)
    assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_activations_over_their_range(act, dtype):
    """Gates from -30 to 30: where the derivatives vanish and where exp would overflow."""
    (x, w_in, w_out), grad = _inputs(96, 48, 56, dtype, seed=3)
    x = (x.float() * 10).to(dtype)
    args = (act, 1.0, 48 ** -0.5, 1.0)
    want = O.gated_feed_forward(x, w_in, w_out, *args, grad, **_roundings(dtype))
    got = _run(x, w_in, w_out, *args, grad)
    for name, value in got.items():
        ref, bound = want[name]
        assert bool(((value.double() - ref).abs() <= bound).all()), name


@pytest.mark.parametrize("n,width,hidden", [(40, 64, 96), (300, 40, 50), (20, 48, 2000)])
def test_gradient_against_differences(n, width, hidden):
    """Central differences of the float32 forward pass along random directions. With steps of 2^-6 the next term of the
    expansion is of relative size 2^-12 times derivatives of order one and the differences keep 6e-8 2^6 of y's size."""
    (x, w_in, w_out), grad = _inputs(n, width, hidden, torch.float32, seed=1)
    args = ("silu", 1.0, width ** -0.5, hidden ** -0.5)
    got = _run(x, w_in, w_out, *args, grad)
    e = 2.0 ** -6
    for k, name in enumerate(NAMES[1:]):
        v = torch.randn_like((x, w_in, w_out)[k])
        v *= math.sqrt(v.numel()) / v.norm() if k == 0 else 1.0
        sides = []
        for s in (e, -e):
            t = [x, w_in, w_out]
            t[k] = t[k] + s * v
            sides.append((_F().gated_feed_forward(*t, *args).double() * grad).sum())
        quotient, exact = float(sides[0] - sides[1]) / (2 * e), float((got[name].double() * v).sum())
        size = float(got[name].double().norm() * v.double().norm())
        assert abs(quotient - exact) <= 2.0 ** -9 * size, name


@pytest.mark.parametrize("dtype", DTYPES)
def test_subsets_of_gradients_and_layouts(dtype):
    """Any subset of the gradients, leading dimensions, strided and unaligned arguments, no rows: as the plain call."""
    (x, w_in, w_out), grad = _inputs(60, 40, 48, dtype, seed=5)
    args = ("gelu", 1.5, 0.2, 0.3)
    full = _run(x, w_in, w_out, *args, grad)
    for mask in range(1, 8):
        leaves = [t.detach().requires_grad_(bool(mask >> k & 1)) for k, t in enumerate((x, w_in, w_out))]
        y = _F().gated_feed_forward(*leaves, *args)
        grads = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], grad)
        names = [n for k, n in enumerate(NAMES[1:]) if mask >> k & 1]
        assert all(torch.equal(g, full[n]) for g, n in zip(grads, names)), mask

    def odd(t):  # the same values one element behind an aligned address
        return torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)

    def strided(t):
        return torch.stack([t, t], dim=-1)[..., 0]

    for f in (odd, strided, lambda t: t.t().contiguous().t()):
        got = _run(f(x), f(w_in), f(w_out), *args, f(grad))
        assert all(torch.equal(got[k], full[k]) for k in full)
    got = _run(x.view(3, 4, 5, 40), w_in, w_out, *args, grad.view(3, 4, 5, 40))
    assert got["y"].shape == (3, 4, 5, 40) and all(torch.equal(got[k].view(full[k].shape), full[k]) for k in full)
    none = _run(x[:0], w_in, w_out, *args, grad[:0])
    assert none["y"].shape == (0, 40) and none["dx"].shape == (0, 40)
    assert not none["dw_in"].any() and not none["dw_out"].any()


# (the last: float32 in three bf16 parts)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,width,hidden", [(70, 48, 80), (4, 260, 70), (700, 24, 16), (8200, 520, 1028)])
def test_values_that_are_not_finite(n, width, hidden, dtype):
    """An infinite or NaN element reaches what the formulas say and nothing else."""
    (x, w_in, w_out), grad = _inputs(n, width, hidden, dtype, seed=2)
    x[1, 3], x[2, 5], w_out[7, 2], grad[3, 1] = math.inf, math.nan, -math.inf, math.inf
    args = ("silu", 1.0, width ** -0.5, hidden ** -0.5)
    want = O.gated_feed_forward(x, w_in, w_out, *args, grad)
    got = _run(x, w_in, w_out, *args, grad)
    for name, value in got.items():
        ref = want[name][0]
        assert torch.equal(value.isnan(), ref.isnan()), name
        assert torch.equal(value == math.inf, ref == math.inf) and torch.equal(value == -math.inf, ref == -math.inf), name


def test_float32_range():
    """float32 operands from 2^-100 to the largest ones keep float32 accuracy."""
    (x, w_in, w_out), grad = _inputs(40, 64, 72, torch.float32, seed=4)
    for sx, si in ((2.0 ** -100, 2.0 ** 97), (2.0 ** 124, 2.0 ** -127)):
        args = ("silu", 1.0, si, 0.1)
        want = O.gated_feed_forward(x * sx, w_in, w_out, *args, None, **_roundings(torch.float32))
        with torch.no_grad():
            _check({"y": _F().gated_feed_forward(x * sx, w_in, w_out, *args)}, want, torch.float32)


def test_refusals():
    F = _F()
    (x, w_in, w_out), _ = _inputs(4, 8, 16, torch.float32)
    with pytest.raises(ValueError, match="act must be one of"):
        F.gated_feed_forward(x, w_in, w_out, "relu")
    with pytest.raises(ValueError, match="are not"):
        F.gated_feed_forward(x, w_in[:30], w_out)
    with pytest.raises(ValueError, match="do not match"):
        F.gated_feed_forward(x[:, :4], w_in, w_out)
    with pytest.raises(TypeError, match="must be"):
        F.gated_feed_forward(x, w_in.half(), w_out)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        F.gated_feed_forward(x, w_in.cpu(), w_out)
    xg = x.clone().requires_grad_(True)
    y = F.gated_feed_forward(xg, w_in, w_out)
    (g,) = torch.autograd.grad(y.square().sum(), xg, create_graph=True)
    with pytest.raises(NotImplementedError, match="second derivatives"):
        torch.autograd.grad(g.sum(), xg)


@pytest.mark.parametrize("dtype", DTYPES)
def test_feed_forward_in_a_graph(dtype):
    """Forward and backward captured on a side stream; every replay, on other inputs, against the eager call."""
    (x, w_in, w_out), grad = _inputs(200, 72, 96, dtype, seed=6)
    leaves = [t.requires_grad_(True) for t in (x, w_in, w_out)]
    args = ("gelu", 1.0, 0.1, 0.1)

    def step():
        y = _F().gated_feed_forward(*leaves, *args)
        return (y.detach(), *torch.autograd.grad(y, leaves, grad))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        with torch.no_grad():
            x.normal_()
            grad.normal_()
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k
