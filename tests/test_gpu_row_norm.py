"""The root-mean-square norm with the residual's addition, its backward pass and its 8-bit form against their float64
statements (``oracle.node_ops.rms_norm_add``, which bounds what a float32 evaluation may be off)."""

import math

import pytest
import torch

from oracle import node_ops as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _F():
    from flashcart_amd.nn import functional as F
    return F


def _inputs(n, width, dtype, seed=0):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    x, res, g, gt = (torch.randn(n, width, device=DEV, generator=gen).to(dtype) for _ in range(4))
    return x, res, (1 + 0.3 * torch.randn(width, device=DEV, generator=gen)).to(dtype), g, gt


def _roundings(dtype):
    return dict(end=torch.finfo(dtype).eps / 2, tiny=2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)


def _check(got, want, dtype):
    for name, value in got.items():
        ref, bound = want[name]
        off = (value.double() - ref).abs()
        assert value.dtype == dtype and value.shape == ref.shape, name
        assert bool((off <= bound).all()), f"{name}: {float((off / bound.clamp_min(1e-300)).max())} times the bound"


def _run(x, res, w, eps, g, gt):
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, res, w)]
    y, total = _F().rms_norm_add(*leaves, eps)
    wanted = [t for t in leaves if t is not None]
    if res is None:
        grads = torch.autograd.grad(y, wanted, g)
    else:
        grads = torch.autograd.grad((y, total), wanted, (g, gt))
    got = {"y": y.detach(), "total": total.detach(), "dx": grads[0]}
    if res is not None:
        assert torch.equal(grads[0], grads[1])
    if w is not None:
        got["dw"] = grads[-1]
    return got


# one element, partial chunks of a lane, every group of lanes, rows that do not fit into registers (backward, both ways),
# more rows than workgroups
SIZES = [(1, 1), (1, 4096), (3, 7), (5, 8), (33, 100), (130, 129), (2000, 128), (1100, 520), (1500, 1031), (3, 5000),
         (1025, 4096), (7, 9001), (5, 12000), (2, 16388), (3, 40003), (1030, 2056), (40000, 20)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,width", SIZES)
def test_norm(n, width, dtype):
    print(f"norm n={n} width={width} {dtype}", flush=True)
    x, res, w, g, gt = _inputs(n, width, dtype)
    for r, weight in ((res, w), (None, w), (res, None)):
        want = O.rms_norm_add(x, r, weight, 1e-5, g, gt if r is not None else None, **_roundings(dtype))
        got = _run(x, r, weight, 1e-5, g, gt)
        _check(got, want, dtype)
        again = _run(x, r, weight, 1e-5, g, gt)
        assert all(torch.equal(got[k], again[k]) for k in got)
        with torch.no_grad():
            y, total = _F().rms_norm_add(x, r, weight, 1e-5)
        assert torch.equal(y, got["y"]) and torch.equal(total, got["total"])


def _check_eight(q, scale, y, slack):
    """Half a step of the 8-bit type off the exact quotient, which `slack` (relative, of y and of the scale) blurs."""
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == torch.float32 and scale.shape == q.shape[:-1]
    _, want = O.e4m3_rows(y)
    assert bool(((scale.double() - want).abs() <= slack * want).all())
    v = y / want[:, None]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    off = (q.double() - v).abs()
    assert bool((off <= step / 2 + 2 * slack * v.abs()).all()), float((off / step).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,width", SIZES)
def test_norm_in_eight_bits(n, width, dtype):
    x, res, w, _, _ = _inputs(n, width, dtype, seed=1)
    slack = (0.25 * width + 8) * 2.0 ** -24
    for r, weight in ((res, w), (None, None)):
        q, scale, total = _F().rms_norm_add_quantized(x, r, weight, 1e-5)
        want = O.rms_norm_add(x, r, weight, 1e-5)
        assert torch.equal(total.double(), want["total"][0])
        _check_eight(q, scale, want["y"][0], slack)
    q, scale = _F().quantize_rows(x)
    _check_eight(q, scale, x.double(), 4 * 2.0 ** -24)


def test_eight_bit_rounding_is_to_nearest_even():
    """Every midpoint between two numbers of the type, its neighbours in float32, and what lies at the type's ends."""
    codes = torch.arange(0, 127, device=DEV, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mid = (codes[1:] + codes[:-1]) / 2
    v = torch.cat([codes, mid, torch.nextafter(mid, mid + 1), torch.nextafter(mid, mid - 1), mid.new_tensor([2.0 ** -12])])
    v = torch.cat([v, -v])
    x = torch.stack([v, torch.flip(v, [0])])  # the largest value is 448: the scale is 1
    q, scale = _F().quantize_rows(x)
    assert torch.equal(scale, torch.ones_like(scale))
    assert torch.equal(q.double(), O.e4m3_rows(x.double())[0])


def test_rows_without_size_and_with_infinities():
    F = _F()
    least = float(torch.tensor(2.0 ** -100 / 448, dtype=torch.float32))
    x = torch.zeros(5, 40, device=DEV)
    x[1, 3], x[2, 5], x[3, 0], x[4] = math.inf, math.nan, 1e-42, 3e38
    y, _ = F.rms_norm_add(x, None, None, 1e-6)
    want = x[0] / math.sqrt(1e-6)
    assert torch.equal(y[0], want) and bool(y[1, 3].isnan()) and not y[1, :3].any() and bool(y[2].isnan().all())
    assert not y[4].any()  # (the squares' sum is infinite, as in float32 it is)
    q, scale = F.quantize_rows(x)
    assert not q[0].float().any() and float(scale[0]) == least
    assert math.isinf(float(scale[1])) and bool(q[1, 3].float().isnan()) and not q[1, :3].float().any()
    assert bool(q[2, 5].float().isnan()) and not q[2, :5].float().any()
    assert not q[3].float().any() and float(scale[3]) == least
    assert bool((q[4].float() == 448).all())
    assert bool(F.rms_norm_add(torch.zeros(2, 8, device=DEV), eps=0.0)[0].isnan().all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_subsets_of_gradients_and_layouts(dtype):
    x, res, w, g, gt = _inputs(60, 40, dtype, seed=5)
    F = _F()
    full = _run(x, res, w, 1e-5, g, gt)
    names = ("dx", "dx", "dw")
    for mask in range(1, 8):
        leaves = [t.detach().requires_grad_(bool(mask >> k & 1)) for k, t in enumerate((x, res, w))]
        y, total = F.rms_norm_add(*leaves, 1e-5)
        # (the total does not depend on the weight)
        outs, cot = ((y, total), (g, gt)) if mask & 3 else ((y,), (g,))
        grads = torch.autograd.grad(outs, [t for t in leaves if t.requires_grad], cot)
        assert all(torch.equal(a, full[names[k]]) for a, k in zip(grads, [k for k in range(3) if mask >> k & 1])), mask
    leaves = [t.detach().requires_grad_(True) for t in (x, res, w)]
    y, total = F.rms_norm_add(*leaves, 1e-5)
    only_y = torch.autograd.grad(y, leaves, g, retain_graph=True)
    assert torch.equal(only_y[2], full["dw"])
    _check({"dx": only_y[0]}, O.rms_norm_add(x, res, w, 1e-5, g, None, **_roundings(dtype)), dtype)
    only_total = torch.autograd.grad(total, leaves, gt, allow_unused=True)
    assert torch.equal(only_total[0], gt) and torch.equal(only_total[1], gt) and only_total[2] is None

    def odd(t):  # the same values one element behind an aligned address
        return torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)

    def strided(t):
        return torch.stack([t, t], dim=-1)[..., 0]

    for f in (odd, strided):
        got = _run(f(x), f(res), f(w), 1e-5, f(g), f(gt))
        assert all(torch.equal(got[k], full[k]) for k in full)
    shaped = (t.view(3, 4, 5, 40) for t in (x, res))
    got = _run(*shaped, w, 1e-5, g.view(3, 4, 5, 40), gt.view(3, 4, 5, 40))
    assert all(torch.equal(got[k].view(full[k].shape), full[k]) for k in full)
    none = _run(x[:0], res[:0], w, 1e-5, g[:0], gt[:0])
    assert none["y"].shape == (0, 40) and none["dx"].shape == (0, 40) and not none["dw"].any()
    q, scale, total = F.rms_norm_add_quantized(x.view(3, 20, 40), res.view(3, 20, 40), w)
    assert q.shape == (3, 20, 40) and scale.shape == (3, 20) and total.shape == (3, 20, 40)
    assert F.quantize_rows(x[:0])[0].shape == (0, 40)


@pytest.mark.parametrize("n,width", [(40, 64), (5, 1031)])
def test_gradient_against_differences(n, width):
    """Central differences of the float32 forward pass along random directions; steps of 2^-6 leave 2^-12 of the next term,
    whose derivatives are of order one, and 2^6 float32 roundings of y."""
    x, res, w, g, gt = _inputs(n, width, torch.float32, seed=2)
    got = _run(x, res, w, 1e-5, g, gt)
    e = 2.0 ** -6
    for k, name in enumerate(("dx", "dx", "dw")):
        gen = torch.Generator(device=DEV).manual_seed(7 + k)
        v = torch.randn((x, res, w)[k].shape, device=DEV, generator=gen)
        sides = []
        for s in (e, -e):
            t = [x, res, w]
            t[k] = t[k] + s * v
            y, total = _F().rms_norm_add(*t, 1e-5)
            sides.append((y.double() * g).sum() + (total.double() * gt).sum())
        quotient, exact = float(sides[0] - sides[1]) / (2 * e), float((got[name].double() * v).sum())
        assert abs(quotient - exact) <= 2.0 ** -9 * float(got[name].double().norm() * v.double().norm()), name


def test_refusals():
    F = _F()
    x, res, w, g, _ = _inputs(4, 8, torch.float32)
    for call in (F.rms_norm_add, F.rms_norm_add_quantized):
        with pytest.raises(ValueError, match="differ in shape"):
            call(x, res[:3], w)
        with pytest.raises(ValueError, match="weight must be"):
            call(x, res, w[:7])
        with pytest.raises(ValueError, match="width 0"):
            call(x[:, :0])
        with pytest.raises(TypeError, match="must be"):
            call(x, res.half(), w)
        with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
            call(x.double())
        with pytest.raises(RuntimeError, match="ROCm devices only"):
            call(x, res.cpu(), w)
    with pytest.raises(NotImplementedError, match="no derivatives"):
        F.rms_norm_add_quantized(x, res, w.clone().requires_grad_())
    with pytest.raises(NotImplementedError, match="no derivatives"):
        F.quantize_rows(x.clone().requires_grad_())
    with torch.no_grad():
        F.rms_norm_add_quantized(x, res, w.clone().requires_grad_())
    xg = x.clone().requires_grad_(True)
    (d,) = torch.autograd.grad(F.rms_norm_add(xg, res, w)[0].square().sum(), xg, create_graph=True)
    with pytest.raises(NotImplementedError, match="second derivatives"):
        torch.autograd.grad(d.sum(), xg)


@pytest.mark.parametrize("dtype", DTYPES)
def test_norm_in_a_graph(dtype):
    """Forward and backward and the 8-bit form captured on a side stream; every replay, on other inputs, as the eager call."""
    x, res, w, g, gt = _inputs(700, 136, dtype, seed=6)
    leaves = [t.requires_grad_(True) for t in (x, res, w)]

    def step():
        y, total = _F().rms_norm_add(*leaves, 1e-5)
        grads = torch.autograd.grad((y, total), leaves, (g, gt))
        with torch.no_grad():
            q, scale, _ = _F().rms_norm_add_quantized(*leaves, 1e-5)
        return (y.detach(), total.detach(), *grads, q.float(), scale)

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
            g.normal_()
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k
