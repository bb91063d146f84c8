"""Dense layers, with one weight and with one for each group of rows, against their float64 statements
(``oracle.node_ops.dense``, which also bounds what the roundings of a float32 evaluation with 16-bit operands may come to,
element by element), and their 8-bit form."""

import math

import pytest
import torch

from oracle import node_ops as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["silu", "sigmoid", "gelu", None]
NAMES = ("y", "dx", "dw", "db", "dres")


def _F():
    from flashcart_amd.nn import functional as F
    return F


def _inputs(n, width, out, dtype, groups=None, seed=0):
    """x, weight, bias, residual, grad"""
    gen = torch.Generator(device=DEV).manual_seed(seed)
    lead = () if groups is None else (groups,)
    return [torch.randn(*s, device=DEV, generator=gen).to(dtype)
            for s in ((n, width), (*lead, out, width), (*lead, out), (n, out), (n, out))]


def _run(x, w, b, res, act, c, s, grad, offsets=None):
    leaves = [t if t is None else t.detach().requires_grad_(True) for t in (x, w, b, res)]
    if offsets is None:
        y = _F().dense(*leaves[:3], act, c, s, leaves[3])
    else:
        y = _F().grouped_dense(leaves[0], leaves[1], offsets, leaves[2], act, c, s)
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], grad)
    return dict(zip([n for n, t in zip(NAMES, (y, *leaves)) if t is not None], (y.detach(), *grads)))


def _roundings(dtype):
    u = torch.finfo(dtype).eps / 2
    if dtype == torch.float32:
        return dict(mid=0.0, end=u, kept=0.0, tiny=2.0 ** -140)
    # The kept derivative holds p = 11 significant bits beside bfloat16, 16 beside float16. A value in [2^k, 2^(k+1)) has steps
    # of 2^(k+1-p), so rounding moves it by up to 2^(k-p), which is 2^-p of it at the lower end: 2^-11 and 2^-16. (Below 2^-14
    # the first is off by up to 2^-25, which the 2^-20 (1 + |z|) of the bound's evaluation of act' holds.)
    return dict(mid=u, end=u, kept=2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -16,
                tiny=2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)


def _check(got, want, dtype):
    # two independent roundings of relative size u, uniform in their interval (u / sqrt 3 each), and the kept derivative;
    # float32: sums in the matrix instructions
    norm = 1e-6 if dtype == torch.float32 else 0.9 * torch.finfo(dtype).eps / 2
    for name, value in got.items():
        if name == "dres":
            continue
        ref, bound = want[name]
        off = (value.double() - ref).abs()
        assert value.dtype == dtype and value.shape == ref.shape, name
        assert bool((off <= bound).all()), f"{name}: {float((off / bound.clamp_min(1e-300)).max())} times the bound"
        if ref.numel() >= 1000:
            assert float(off.norm()) <= norm * float(ref.norm()), f"{name}: relative error {float(off.norm() / ref.norm())}"


# one row, sizes of one, odd ones, more than one tile each way, long sums of few outputs, every tile size with and without
# ragged edges, few rows at which the forward pass has kernels of its own
SIZES = [(1, 1, 1), (1, 64, 64), (1, 4096, 520), (3, 5, 7), (17, 33, 19), (64, 128, 512), (130, 96, 200), (257, 519, 103),
         (1000, 64, 72), (5, 2056, 40), (70, 40, 3001), (9001, 24, 16), (2049, 136, 264), (4096, 512, 1024),
         (4100, 520, 1100), (16, 1024, 2048), (48, 2048, 1000), (33, 72, 4099), (9, 100, 2056), (8200, 520, 1032)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,width,out", SIZES)
def test_dense(n, width, out, dtype):
    act = ACTS[(n + width + out) % 4]
    print(f"dense n={n} width={width} out={out} {act} {dtype}", flush=True)
    x, w, b, res, grad = _inputs(n, width, out, dtype)
    args = (act, 1.6, width ** -0.5)
    for bias, residual in ((b, res), (None, None)):
        want = O.dense(x, w, bias, residual, *args, grad, **_roundings(dtype))
        got = _run(x, w, bias, residual, *args, grad)
        _check(got, want, dtype)
        if residual is not None:
            assert torch.equal(got["dres"], grad)
        with torch.no_grad():
            _check({"y": _F().dense(x, w, bias, *args, residual)}, want, dtype)
        again = _run(x, w, bias, residual, *args, grad)
        assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_activations_over_their_range(act, dtype):
    """Arguments from -30 to 30: where the derivatives vanish and where exp would overflow."""
    x, w, b, res, grad = _inputs(96, 48, 56, dtype, seed=3)
    x = (x.float() * 10).to(dtype)
    args = (act, 1.0, 48 ** -0.5)
    want = O.dense(x, w, b, None, *args, grad, **_roundings(dtype))
    got = _run(x, w, b, None, *args, grad)
    for name, value in got.items():
        ref, bound = want[name]
        assert bool(((value.double() - ref).abs() <= bound).all()), name


def _offsets(counts, first=0, dtype=torch.int64):
    return torch.tensor([first, *counts], device=DEV).cumsum(0).to(dtype)


# rows of each group, rows in front of the first and behind the last: one row, empty groups, one group, more groups than lanes,
# groups of partial tiles, sums over rows in one part and in several
GROUPS = [(1, 1, 1, [1], 0, 0), (5, 7, 9, [0, 3, 0, 1, 0], 1, 2), (33, 40, 16, [0, 0, 0], 2, 1), (64, 128, 64, [70, 0, 64, 1], 0, 0),
          (24, 48, 40, [k % 5 for k in range(150)], 3, 40), (136, 72, 264, [300, 5, 900, 64, 0, 31], 0, 7),
          (520, 264, 328, [1000, 20, 2000, 4], 0, 0), (128, 128, 128, [6000, 7000, 100, 5900], 0, 0),
          (2048, 520, 1000, [2, 0, 1, 9, 0, 0, 4, 1], 0, 3), (264, 520, 1032, [8, 2000, 0, 6000], 5, 0),
          (600, 512, 512, [5000, 5000], 0, 0), (16, 16, 24, [0] * 63 + [5] + [0] * 70 + [2], 0, 0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", range(len(GROUPS)))
def test_grouped_dense(case, dtype):
    _, width, out, counts, front, back = GROUPS[case]
    n, act = front + sum(counts) + back, ACTS[case % 4]
    print(f"grouped width={width} out={out} {counts[:8]} {act} {dtype}", flush=True)
    x, w, b, _, grad = _inputs(n, width, out, dtype, groups=len(counts))
    offsets = _offsets(counts, front, torch.int32 if case % 2 else torch.int64)
    args = (act, 1.6, width ** -0.5)
    for bias in (b, None):
        want = O.grouped_dense(x.cpu(), w.cpu(), offsets.cpu(), None if bias is None else bias.cpu(), *args, grad.cpu(),
                               **_roundings(dtype))
        want = {k: tuple(t.to(DEV) for t in v) for k, v in want.items()}
        got = _run(x, w, bias, None, *args, grad, offsets)
        _check(got, want, dtype)
        with torch.no_grad():
            _check({"y": _F().grouped_dense(x, w, offsets, bias, *args)}, want, dtype)
        again = _run(x, w, bias, None, *args, grad, offsets)
        assert all(torch.equal(got[k], again[k]) for k in got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
def test_gradients_of_short_groups(act, dtype):
    """The bias' gradients of one to three rows, some of which cancel: what is left is off by the kept derivatives' rounding."""
    counts = [1, 2, 3] * 10
    x, w, b, _, grad = _inputs(sum(counts), 21, 896, dtype, groups=len(counts), seed=4)
    offsets, args = _offsets(counts), (act, 1.0, 21 ** -0.5)
    want = O.grouped_dense(*(t.cpu() for t in (x, w, offsets, b)), *args, grad.cpu(), **_roundings(dtype))
    _check(_run(x, w, b, None, *args, grad, offsets), {k: tuple(t.to(DEV) for t in v) for k, v in want.items()}, dtype)


@pytest.mark.parametrize("offsets", [[-5, 3, 2, 100, 7], [9, 9, 4, 4, 200], [50, 60, 70, 80, 90], [-9, -8, -7, -6, -1],
                                     [-2 ** 62, 2 ** 62, 0, 5, -3], [3, 20, 20, 11, 33]])
def test_offsets_of_any_value(offsets):
    """They are taken into the rows and as their running maximum."""
    x, w, b, _, grad = _inputs(40, 24, 32, torch.float32, groups=4, seed=4)
    off = torch.tensor(offsets, device=DEV)
    want = O.grouped_dense(x.cpu(), w.cpu(), off.cpu(), b.cpu(), "silu", 1.0, 0.2, grad.cpu(), **_roundings(torch.float32))
    got = _run(x, w, b, None, "silu", 1.0, 0.2, grad, off)
    _check(got, {k: tuple(t.to(DEV) for t in v) for k, v in want.items()}, torch.float32)


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("n,width,out", [(1, 16, 16), (3, 5, 7), (17, 33, 19), (64, 128, 512), (257, 519, 103), (5, 2056, 40),
                                         (9, 4096, 520), (48, 2048, 1000), (2049, 144, 264), (4100, 1024, 1100), (70, 8192, 64)])
def test_quantized_dense(n, width, out, dtype):
    """Against float64 products of the same 8-bit numbers. The instruction adds the products of 8 k with 13 bits below the
    leading bit of the largest, so that each may lose 2^-13 of that."""
    act = ACTS[(n + width + out) % 4]
    x, w, b, res, _ = _inputs(n, width, out, dtype, seed=1)
    (qx, sx), (qw, sw) = _F().quantize_rows(x), _F().quantize_rows(w)
    xv, wv = qx.double() * sx.double()[:, None], qw.double() * sw.double()[:, None]
    for bias, residual in ((b, res), (None, None)):
        y, bound = O.dense(xv, wv, bias, residual, act, 1.6, width ** -0.5, **_roundings(dtype))["y"]
        got = _F().quantized_dense(qx, sx, qw, sw, bias, act, 1.6, width ** -0.5, residual, dtype)
        most = (xv.abs().amax(1)[:, None] * wv.abs().amax(1)) * width * 2.0 ** -13 * width ** -0.5 * 1.6 * 1.13
        off = (got.double() - y).abs()
        assert y.numel() < 1000 or float(off.norm()) <= 0.9 * torch.finfo(dtype).eps / 2 * float(y.norm())
        assert got.dtype == dtype and got.shape == y.shape
        assert bool((off <= bound + most).all()), float((off / (bound + most)).max())
        again = _F().quantized_dense(qx, sx, qw, sw, bias, act, 1.6, width ** -0.5, residual, dtype)
        assert torch.equal(got, again)


@pytest.mark.parametrize("dtype", DTYPES[1:])
def test_every_eight_bit_number_in_a_product(dtype):
    """Each number of the type times one, in every place of a row: exact."""
    v = torch.arange(256, device=DEV, dtype=torch.int32).to(torch.uint8)
    v = v[(v & 127) != 127].view(torch.float8_e4m3fn)
    x = torch.zeros(v.numel(), 272, device=DEV)
    at = torch.arange(v.numel(), device=DEV)
    x[at, at] = v.float()
    one = torch.ones(v.numel(), device=DEV)
    eye = torch.eye(272, device=DEV).to(torch.float8_e4m3fn)
    y = _F().quantized_dense(x.to(torch.float8_e4m3fn), one, eye, torch.ones(272, device=DEV), dtype=dtype)
    assert torch.equal(y.float(), x)


@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("n,width,out", [(40, 64, 96), (300, 40, 50), (20, 48, 2000)])
def test_gradient_against_differences(n, width, out, grouped):
    """Central differences of the float32 forward pass along random directions: steps of 2^-6 leave 2^-12 of the next term,
    with derivatives of order one, and 2^6 float32 roundings of y."""
    x, w, b, res, grad = _inputs(n, width, out, torch.float32, groups=3 if grouped else None, seed=1)
    offsets = _offsets([n // 2, 0, n // 3]) if grouped else None
    if grouped:
        res = None
    args = ("silu", 1.0, width ** -0.5)
    got = _run(x, w, b, res, *args, grad, offsets)
    e = 2.0 ** -6
    for k, name in enumerate(NAMES[1:4]):
        gen = torch.Generator(device=DEV).manual_seed(7 + k)
        v = torch.randn((x, w, b)[k].shape, device=DEV, generator=gen)
        sides = []
        for s in (e, -e):
            t = [x, w, b]
            t[k] = t[k] + s * v
            y = _F().grouped_dense(t[0], t[1], offsets, t[2], *args) if grouped else _F().dense(*t, *args, res)
            sides.append((y.double() * grad).sum())
        quotient, exact = float(sides[0] - sides[1]) / (2 * e), float((got[name].double() * v).sum())
        assert abs(quotient - exact) <= 2.0 ** -9 * float(got[name].double().norm() * v.double().norm()), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("grouped", [False, True])
def test_subsets_of_gradients_and_layouts(grouped, dtype):
    """Any subset of the gradients, leading dimensions, strided and unaligned arguments, no rows: as the plain call."""
    x, w, b, res, grad = _inputs(60, 40, 48, dtype, groups=3 if grouped else None, seed=5)
    offsets = _offsets([20, 0, 38], 1) if grouped else None
    res = None if grouped else res
    args = ("gelu", 1.5, 0.2)
    full = _run(x, w, b, res, *args, grad, offsets)
    tensors = (x, w, b) if grouped else (x, w, b, res)
    for mask in range(1, 1 << len(tensors)):
        leaves = [t.detach().requires_grad_(bool(mask >> k & 1)) for k, t in enumerate(tensors)]
        if grouped:
            y = _F().grouped_dense(leaves[0], leaves[1], offsets, leaves[2], *args)
        else:
            y = _F().dense(*leaves[:3], *args, leaves[3])
        grads = torch.autograd.grad(y, [t for t in leaves if t.requires_grad], grad)
        names = [n for k, n in enumerate(NAMES[1:]) if mask >> k & 1]
        assert all(torch.equal(g, full[n]) for g, n in zip(grads, names)), mask

    def odd(t):  # the same values one element behind an aligned address
        return torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape)

    def strided(t):
        return torch.stack([t, t], dim=-1)[..., 0]

    for f in (odd, strided, lambda t: t.transpose(0, -1).contiguous().transpose(0, -1)):
        got = _run(f(x), f(w), f(b), None if grouped else f(res), *args, f(grad), offsets)
        assert all(torch.equal(got[k], full[k]) for k in full)
    if not grouped:
        got = _run(x.view(3, 4, 5, 40), w, b, res.view(3, 4, 5, 48), *args, grad.view(3, 4, 5, 48))
        assert got["y"].shape == (3, 4, 5, 48) and all(torch.equal(got[k].view(full[k].shape), full[k]) for k in full)
    none = _run(x[:0], w, b, None if grouped else res[:0], *args, grad[:0], offsets)
    assert none["y"].shape == (0, 48) and none["dx"].shape == (0, 40) and not none["dw"].any() and not none["db"].any()


# (the last: float32 in three bf16 parts)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("n,width,out", [(70, 48, 80), (4, 260, 70), (700, 24, 16), (8200, 520, 1028)])
def test_values_that_are_not_finite(n, width, out, grouped, dtype):
    """An infinite or NaN element reaches what the formulas say and nothing else."""
    x, w, b, _, grad = _inputs(n, width, out, dtype, groups=2 if grouped else None, seed=2)
    x[1, 3], x[2, 5], grad[3, 1] = math.inf, math.nan, math.inf
    (w[1] if grouped else w)[7, 2] = -math.inf
    args = ("silu", 1.0, width ** -0.5)
    offsets = _offsets([n // 2, n - n // 2]) if grouped else None
    if grouped:
        want = O.grouped_dense(x.cpu(), w.cpu(), offsets.cpu(), b.cpu(), *args, grad.cpu())
        want = {k: tuple(t.to(DEV) for t in v) for k, v in want.items()}
    else:
        want = O.dense(x, w, b, None, *args, grad)
    got = _run(x, w, b, None, *args, grad, offsets)
    for name, value in got.items():
        ref = want[name][0]
        assert torch.equal(value.isnan(), ref.isnan()), name
        assert torch.equal(value == math.inf, ref == math.inf) and torch.equal(value == -math.inf, ref == -math.inf), name


def test_float32_range():
    """float32 operands from 2^-100 to the largest ones keep float32 accuracy."""
    x, w, b, _, _ = _inputs(40, 64, 72, torch.float32, seed=4)
    for sx, s in ((2.0 ** -100, 2.0 ** 97), (2.0 ** 124, 2.0 ** -127)):
        want = O.dense(x * sx, w, b, None, "silu", 1.0, s, **_roundings(torch.float32))
        with torch.no_grad():
            _check({"y": _F().dense(x * sx, w, b, "silu", 1.0, s)}, want, torch.float32)


def test_refusals():
    F = _F()
    x, w, b, res, _ = _inputs(4, 8, 16, torch.float32)
    with pytest.raises(ValueError, match="act must be None or one of"):
        F.dense(x, w, b, "relu")
    with pytest.raises(ValueError, match="do not match"):
        F.dense(x[:, :4], w)
    with pytest.raises(ValueError, match="weight must be"):
        F.dense(x, w[0])
    with pytest.raises(ValueError, match="not empty"):
        F.dense(x, w[:0])
    with pytest.raises(ValueError, match="bias must be"):
        F.dense(x, w, b[:3])
    with pytest.raises(ValueError, match="residual must be"):
        F.dense(x, w, residual=res[:3])
    with pytest.raises(TypeError, match="must be"):
        F.dense(x, w.half())
    with pytest.raises(TypeError, match="float32, bfloat16 or float16"):
        F.dense(x.double(), w.double())
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        F.dense(x, w.cpu())
    off = _offsets([1, 3])
    w2 = torch.stack([w, w])
    with pytest.raises(ValueError, match="offsets must be"):
        F.grouped_dense(x, w2, off[:2])
    with pytest.raises(TypeError, match="int64 or int32"):
        F.grouped_dense(x, w2, off.float())
    with pytest.raises(TypeError, match="must be a tensor"):
        F.grouped_dense(x, w2, None)
    with pytest.raises(ValueError, match="weight must be"):
        F.grouped_dense(x, w, off)
    with pytest.raises(ValueError, match="bias must be"):
        F.grouped_dense(x, w2, off, b)
    with pytest.raises(ValueError, match="do not match"):
        F.grouped_dense(x.view(2, 2, 8), w2, off)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        F.grouped_dense(x, w2, off.cpu())
    (qx, sx), (qw, sw) = F.quantize_rows(x), F.quantize_rows(w)
    with pytest.raises(TypeError, match="must be"):
        F.quantized_dense(x, sx, qw, sw)
    with pytest.raises(ValueError, match="one for each row"):
        F.quantized_dense(qx, sx[:2], qw, sw)
    with pytest.raises(TypeError, match="dtype"):
        F.quantized_dense(qx, sx, qw, sw, dtype=torch.float32)
    with pytest.raises(TypeError, match="must be"):
        F.quantized_dense(qx, sx, qw, sw, b, dtype=torch.bfloat16)
    with pytest.raises(NotImplementedError, match="no derivatives"):
        F.quantized_dense(qx, sx, qw, sw, b.bfloat16().requires_grad_())
    xg = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(F.dense(xg, w, b, "silu").square().sum(), xg, create_graph=True)
    with pytest.raises(NotImplementedError, match="second derivatives"):
        torch.autograd.grad(g.sum(), xg)


@pytest.mark.parametrize("dtype", DTYPES)
def test_dense_layers_in_a_graph(dtype):
    """Forward and backward captured on a side stream; every replay, on other inputs and groups, as the eager call."""
    x, w, b, res, grad = _inputs(200, 72, 96, dtype, seed=6)
    _, wg, bg, _, _ = _inputs(200, 96, 72, dtype, groups=3, seed=7)
    leaves = [t.requires_grad_(True) for t in (x, w, b, res, wg, bg)]
    offsets = _offsets([50, 100, 50])
    F = _F()

    def step():
        y = F.dense(*leaves[:3], "gelu", 1.0, 0.1, leaves[3])
        z = F.grouped_dense(y, leaves[4], offsets, leaves[5], "silu", 1.0, 0.1)
        grads = torch.autograd.grad(z, leaves, grad[:, :72])
        with torch.no_grad():
            eight = F.quantized_dense(*F.quantize_rows(x), *F.quantize_rows(w), b.bfloat16())
        return (z.detach(), *grads, eight)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.current_stream().wait_stream(side)
    for k, counts in enumerate(([50, 100, 50], [0, 200, 0], [1, 2, 3], [199, 0, 1])):
        with torch.no_grad():
            x.normal_()
            grad.normal_()
            offsets.copy_(_offsets(counts))
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k
