"""Dense layers where their values are hard to hold: infinite arguments of every activation, derivatives that vanish."""

import math

import pytest
import torch

from oracle import node_ops as O
from tests.test_gpu_dense import ACTS, DEV, DTYPES, _check, _F, _inputs, _offsets, _roundings, _run

pytestmark = pytest.mark.gpu


# tiles of 64 rows, few rows, sums in parts, rows that are not whole chunks, float32 in three bf16 parts
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("grouped", [False, True])
@pytest.mark.parametrize("n,width,out", [(70, 48, 80), (4, 256, 72), (64, 4096, 64), (300, 45, 53), (8200, 520, 1032)])
def test_infinite_biases(n, width, out, grouped, act, dtype):
    """A bias of -inf or inf: the logistic function is 0 or 1 there with a derivative of 0, so that the other columns keep
    their gradients; elsewhere what the formulas say."""
    print(f"infinite biases n={n} width={width} out={out} {act} {dtype} grouped={grouped}", flush=True)
    x, w, b, _, grad = _inputs(n, width, out, dtype, groups=2 if grouped else None, seed=8)
    b[..., 3], b[..., 5], b[..., out - 1], b[..., 6] = -math.inf, math.inf, -math.inf, math.nan
    args = (act, 1.5, width ** -0.5)
    keep = torch.ones(out, dtype=torch.bool, device=DEV)
    keep[[3, 5, 6, out - 1]] = False
    offsets = _offsets([n // 2, n - n // 2]) if grouped else None

    def oracle(x, w, b, grad):
        if not grouped:
            return O.dense(x, w, b, None, *args, grad, **_roundings(dtype))
        want = O.grouped_dense(x.cpu(), w.cpu(), offsets.cpu(), b.cpu(), *args, grad.cpu(), **_roundings(dtype))
        return {k: tuple(t.to(DEV) for t in v) for k, v in want.items()}

    got = _run(x, w, b, None, *args, grad, offsets)
    want = oracle(x, w, b, grad)["y"][0]
    for p in (math.inf, -math.inf):
        assert torch.equal(got["y"] == p, want == p)
    assert torch.equal(got["y"].isnan(), want.isnan())
    if act == "sigmoid":
        assert not got["y"][:, 3].any() and bool((got["y"][:, 5] == torch.tensor(1.5, dtype=dtype)).all())
        assert not got["db"][..., [3, 5, out - 1]].any() and not got["dw"][..., [3, 5, out - 1], :].any()
    rest = oracle(x, w[..., keep, :], b[..., keep], grad[:, keep])
    _check({"y": got["y"][:, keep], "dw": got["dw"][..., keep, :], "db": got["db"][..., keep]}, rest, dtype)
    # without the NaN, whose column every row of dx has a part of
    b[..., 6] = -math.inf
    if act == "sigmoid":
        got = _run(x, w, b, None, *args, grad, offsets)
        _check({"dx": got["dx"]}, rest, dtype)


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("n,width,out", [(1, 64, 80), (40, 2048, 80), (300, 400, 530)])
def test_infinite_biases_in_eight_bits(n, width, out, act, dtype):
    x, w, b, _, _ = _inputs(n, width, out, dtype, seed=9)
    b[3], b[5], b[6] = -math.inf, math.inf, math.nan
    (qx, sx), (qw, sw) = _F().quantize_rows(x), _F().quantize_rows(w)
    got = _F().quantized_dense(qx, sx, qw, sw, b, act, 1.5, width ** -0.5, dtype=dtype)
    want = O.dense(qx.double() * sx.double()[:, None], qw.double() * sw.double()[:, None], b, None, act, 1.5, width ** -0.5)["y"][0]
    for p in (math.inf, -math.inf):
        assert torch.equal(got == p, want == p)
    assert torch.equal(got.isnan(), want.isnan())
    if act == "sigmoid":
        assert not got[:, 3].any() and bool((got[:, 5] == torch.tensor(1.5, dtype=dtype)).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_sums_that_leave_the_range(dtype):
    """Sums beyond float32: gates that are closed or open altogether, with no gradient."""
    n, width, out = 40, 64, 72
    most = float(torch.finfo(dtype).max)
    x, w = torch.full((n, width), most, device=DEV, dtype=dtype), torch.full((out, width), most, device=DEV, dtype=dtype)
    w[::2] *= -1
    s = 3e38 if dtype == torch.float16 else 1.0
    grad = torch.ones(n, out, device=DEV, dtype=dtype)
    got = _run(x, w, None, None, "sigmoid", 1.0, s, grad)
    assert not got["y"][:, ::2].any() and bool((got["y"][:, 1::2] == 1).all()) and not got["dw"].any()


# activation and the range of its argument
RANGES = [("silu", -40.0, 40.0), ("sigmoid", -40.0, 40.0), ("gelu", -14.0, 14.0)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,low,high", RANGES)
@pytest.mark.parametrize("n", [1, 70, 300])
def test_derivatives_that_vanish(n, act, low, high, dtype):
    """act'(z) through the bias' gradient of one row, relative to itself: one rounding of the type (eps / 2), the kept
    derivative's (2^-11 beside bfloat16, with float16's smallest half step 2^-25 after a factor of 2^15, so 2^-40; 2^-16 beside
    float16), and what float32 makes of the formula: 8 roundings of its terms, and an exponential whose argument, rounded, is off
    by 2^-24 of itself. exp(-z^2 / 2) is below float32's smallest normal number 2^-126 from |z| = 13.22 on, where the
    exponential instruction gives zero: an error of that, times R + |z| pdf(0) <= 0.5 + 14 x 0.4 < 2^3, in gelu's."""
    print(f"derivatives n={n} {act} {dtype}", flush=True)
    z = torch.linspace(low, high, 1000, device=DEV).to(dtype)
    x, w = torch.zeros(n, 8, device=DEV, dtype=dtype), torch.randn(1000, 8, device=DEV).to(dtype)
    grad = torch.zeros(n, 1000, device=DEV, dtype=dtype)
    grad[n // 2] = 1
    got = _run(x, w, z, None, act, 1.0, 1.0, grad)
    v = z.double()
    s = torch.sigmoid(v)
    t = torch.sigmoid(-v)  # 1 - s
    if act == "gelu":
        cdf, pdf = 0.5 * torch.erfc(-v / math.sqrt(2)), torch.exp(-0.5 * v * v) / math.sqrt(2 * math.pi)
        want = cdf + v * pdf
        terms = (cdf + v.abs() * pdf) * (1 + v * v)
    elif act == "sigmoid":
        want = s * t
        terms = want * (1 + v.abs())
    else:
        want = s * (1 + v * t)
        terms = s * (1 + v.abs() * t) * (1 + v.abs())
    u = torch.finfo(dtype).eps / 2
    kept, least = {torch.float32: (0.0, 0.0), torch.bfloat16: (2.0 ** -11, 2.0 ** -40),
                   torch.float16: (2.0 ** -16, 0.0)}[dtype]
    bound = (u + kept + u * kept) * want.abs() + least + 8 * 2.0 ** -24 * terms
    bound = bound + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -123 if act == "gelu" else 2.0 ** -134)
    off = (got["db"].double() - want).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), float(z[(off / bound).argmax()]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 70, 300])
def test_tails_of_gelu(n, dtype):
    """y relative to itself: one rounding of the type, 8 of float32, and those of the exponential's argument."""
    z = torch.linspace(-13, 13, 1000, device=DEV).to(dtype)
    x, w = torch.zeros(n, 8, device=DEV, dtype=dtype), torch.randn(1000, 8, device=DEV).to(dtype)
    v = z.double()
    want = 0.5 * v * torch.erfc(-v / math.sqrt(2))
    bound = (torch.finfo(dtype).eps / 2 + 8 * 2.0 ** -24 * (1 + v * v)) * want.abs()
    bound = bound + (2.0 ** -25 if dtype == torch.float16 else 2.0 ** -134)
    off = (_F().dense(x, w, z, "gelu").double() - want).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), float(z[(off / bound).amax(0).argmax()]))


@pytest.mark.parametrize("dtype", DTYPES[:2])
def test_large_gradients(dtype):
    """Gradients near the largest number of the type, whose product with the activation's factor alone would leave it: silu'(0) =
    1/2, so the bias' gradient is exactly 5/6 of it."""
    n, out = 40, 72
    x, w, z = (torch.zeros(*s, device=DEV, dtype=dtype) for s in ((n, 8), (out, 8), (out,)))
    grad = torch.zeros(n, out, device=DEV, dtype=dtype)
    grad[17] = 1.5 * 2.0 ** 127
    got = _run(x, w, z, None, "silu", 5 / 3, 1.0, grad)
    want = grad[17].double() * float(torch.tensor(5 / 3, dtype=torch.float32)) / 2
    off = (got["db"].double() - want).abs()
    assert bool((off <= (torch.finfo(dtype).eps / 2 + 2.0 ** -23) * want).all())
