"""The 8-bit numbers of the row norm and of rows themselves, number by number: for 16-bit values 448 t w / max|t w| is stated in
float64 without an error that matters, its midpoints between two e4m3 numbers among it."""

import math

import pytest
import torch

from tests.test_gpu_row_norm import DEV, _F, _inputs

pytestmark = pytest.mark.gpu
HALF = [torch.bfloat16, torch.float16]
# every group of lanes, partial chunks, rows that do not fit into registers
SIZES = [(3, 7), (500, 100), (300, 520), (60, 1031), (100, 5000), (9, 16392), (5, 40003)]


def _nearest(v):
    """(nearest e4m3 numbers, ties to even; whether v is a midpoint) of |v| <= 448 in float64. v is rounded to float32 first,
    which has every midpoint, and never moves a value across one."""
    v = v.float().double()
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(v / step) * step, (v / step).frac().abs() == 0.5


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("n,width", SIZES)
def test_every_number_is_the_nearest(n, width, dtype):
    """Products t w of 16-bit values and 448 times them are exact in float64, so a midpoint comes out as one."""
    x, res, w, _, _ = _inputs(n, width, dtype, seed=11)
    total = (x.float() + res.float()).to(dtype)
    for r, weight, t in ((res, w, total), (None, w, x), (None, None, x)):
        p = t.double() * (1 if weight is None else weight.double())
        want, middle = _nearest(448 * p / p.abs().amax(1, keepdim=True))
        # (one in 8,000 quotients of products of 8-bit significands is a midpoint; of 11-bit ones, 2^6 times fewer)
        assert n * width < 30000 or dtype == torch.float16 or bool(middle.any())
        got = _F().rms_norm_add_quantized(x, r, weight, 1e-5)[0]
        assert torch.equal(got.double(), want), int((got.double() != want).sum())
    want, _ = _nearest(448 * x.double() / x.double().abs().amax(1, keepdim=True))
    assert torch.equal(_F().quantize_rows(x)[0].double(), want)


@pytest.mark.parametrize("dtype", [torch.float32, *HALF])
def test_rows_of_every_size(dtype):
    """Rows from the smallest to the largest numbers: nearest while the row's largest value is above 2^-100; below, that least
    scale, under which all values round to zero or the few smallest numbers."""
    gen = torch.Generator(device=DEV).manual_seed(12)
    low, high = (-14, 15) if dtype == torch.float16 else (-126, 127)
    rows = torch.arange(low, high + 1, device=DEV, dtype=torch.float64)
    x = (torch.rand(rows.numel(), 200, device=DEV, generator=gen, dtype=torch.float64) * 2 - 1) * torch.exp2(rows)[:, None]
    x = x.to(dtype)
    q, scale = _F().quantize_rows(x)
    v = x.double()
    most = v.abs().amax(1, keepdim=True)
    top = most.clamp_min(2.0 ** -100)
    assert bool(((scale.double() - top[:, 0] / 448).abs() <= 2.0 ** -24 * top[:, 0] / 448).all())
    want, _ = _nearest(448 * v / top)
    exact = (most >= 2.0 ** -100).expand_as(v) if dtype != torch.float32 else torch.zeros_like(v, dtype=torch.bool)
    assert torch.equal(q.double()[exact], want[exact])
    # half a step, of the quotient by a scale that was rounded (2^-24) and by float32's rounding of it
    step = torch.exp2(torch.floor(torch.log2((448 * v / top).abs().clamp_min(2.0 ** -6))) - 3)
    off = (q.double() - 448 * v / top).abs()
    assert bool((off <= step / 2 + 2.0 ** -23 * (448 * v / top).abs()).all())


def test_norms_of_rows_with_infinities():
    """The sum of squares is infinite, so every finite value's norm is zero; the infinity itself has none. A NaN is in all of
    its row's values."""
    x = torch.randn(4, 40, device=DEV)
    x[1, 3], x[2, 5], x[3] = math.inf, math.nan, 3e38
    q, scale, _ = _F().rms_norm_add_quantized(x, None, None, 1e-6)
    y = q.double() * scale.double()[:, None]
    least = float(torch.tensor(2.0 ** -100 / 448, dtype=torch.float32))
    assert bool(y[1, 3].isnan()) and not y[1, :3].any() and not y[1, 4:].any() and float(scale[1]) == least
    assert bool(y[2].isnan().all())
    assert not y[3].any() and float(scale[3]) == least
    # a weight with an infinity: there the norm is infinite, and the row's scale
    w = torch.ones(40, device=DEV)
    w[7] = -math.inf
    q, scale, _ = _F().rms_norm_add_quantized(x[:1], None, w, 1e-6)
    assert math.isinf(float(scale)) and bool(q[0, 7].float().isnan()) and not q[0, :7].float().any()
