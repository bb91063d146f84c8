"""Dense layers at sizes that take the largest output tiles, with a last round of them in two halves, ragged rows and columns:
every part of the epilogue, and all gradients. Each test asserts that its size takes those tiles."""

import ctypes

import pytest
import torch

from oracle import node_ops as O
from tests.test_gpu_dense import DEV, DTYPES, _check, _F, _inputs, _offsets, _roundings, _run

pytestmark = pytest.mark.gpu


def _tile(dtype, n, width, out, groups=0, act=0, which=0):
    from flashcart_amd import _lib
    halves = ctypes.c_int32(-1)
    desc = _lib.DenseDesc(DTYPES.index(dtype), act, width, out, groups, 1, 1.0, 1.0)
    return _lib.load().fc_node_dense_tile(desc, n, which, halves), halves.value


@pytest.fixture(autouse=True)
def _memory_is_given_back():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


# whole chunks of 16 bytes, and rows that are copied
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,width,out,act", [(4360, 2056, 4872, "silu"), (4357, 2051, 4869, "gelu"), (4360, 2056, 4872, None)])
def test_dense(n, width, out, act, dtype):
    print(f"dense n={n} width={width} out={out} {act} {dtype}", flush=True)
    assert _tile(dtype, n, width, out) == (256, 104) and _tile(dtype, n, width, out, which=2)[0] == 256
    x, w, b, res, grad = _inputs(n, width, out, dtype, seed=20)
    args = (act, 1.6, width ** -0.5)
    for bias, residual in ((b, res), (None, None)):
        want = O.dense(x, w, bias, residual, *args, grad, **_roundings(dtype))
        got = _run(x, w, bias, residual, *args, grad)
        _check(got, want, dtype)
        again = _run(x, w, bias, residual, *args, grad)
        assert all(torch.equal(got[k], again[k]) for k in got)
        with torch.no_grad():
            assert torch.equal(_F().dense(x, w, bias, *args, residual), got["y"])


@pytest.mark.parametrize("dtype", DTYPES[1:])
@pytest.mark.parametrize("n,width,out,act", [(4360, 4112, 4872, "silu"), (4357, 4109, 4869, None), (8200, 4096, 4112, "gelu")])
def test_quantized_dense(n, width, out, act, dtype):
    """The bound is that of the smaller sizes' test: each of 8 products may lose 2^-13 of the largest."""
    print(f"8 bits n={n} width={width} out={out} {act} {dtype}", flush=True)
    tile, halves = _tile(dtype, n, width, out, which=1)
    assert tile == 256 and halves == (104 if n < 5000 else 49)
    x, w, b, res, _ = _inputs(n, width, out, dtype, seed=21)
    (qx, sx), (qw, sw) = _F().quantize_rows(x), _F().quantize_rows(w)
    xv, wv = qx.double() * sx.double()[:, None], qw.double() * sw.double()[:, None]
    for bias, residual in ((b, res), (None, None)):
        y, bound = O.dense(xv, wv, bias, residual, act, 1.6, width ** -0.5, **_roundings(dtype))["y"]
        got = _F().quantized_dense(qx, sx, qw, sw, bias, act, 1.6, width ** -0.5, residual, dtype)
        most = (xv.abs().amax(1)[:, None] * wv.abs().amax(1)) * width * 2.0 ** -13 * width ** -0.5 * 1.6 * 1.13
        off = (got.double() - y).abs()
        assert float(off.norm()) <= 0.9 * torch.finfo(dtype).eps / 2 * float(y.norm())
        assert bool((off <= bound + most).all()), float((off / (bound + most)).max())
        assert torch.equal(got, _F().quantized_dense(qx, sx, qw, sw, bias, act, 1.6, width ** -0.5, residual, dtype))


# uneven groups, some without rows, rows of none; sums over rows in one part
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width,out,counts,front,back,act", [(2056, 2056, [2500, 3, 0, 3300], 2, 195, "silu"),
                                                             (2565, 2051, [100, 5700], 0, 200, "sigmoid")])
def test_grouped_dense(width, out, counts, front, back, act, dtype):
    n, groups = front + sum(counts) + back, len(counts)
    print(f"grouped width={width} out={out} {counts} {act} {dtype}", flush=True)
    assert _tile(dtype, n, width, out, groups)[0] == 256 and _tile(dtype, n, width, out, groups, which=2)[0] == 256
    x, w, b, _, grad = _inputs(n, width, out, dtype, groups=groups, seed=22)
    offsets, args = _offsets(counts, front), (act, 1.6, width ** -0.5)
    got = _run(x, w, b, None, *args, grad, offsets)
    for name in ("y", "dx"):
        assert not got[name][:front].any() and not got[name][n - back:].any()
    for e, (p, q) in enumerate(O.group_rows(offsets, n)):
        want = O.dense(x[p:q], w[e], b[e], None, *args, grad[p:q], **_roundings(dtype))
        _check({"y": got["y"][p:q], "dx": got["dx"][p:q], "dw": got["dw"][e], "db": got["db"][e]}, want, dtype)
    again = _run(x, w, b, None, *args, grad, offsets)
    assert all(torch.equal(got[k], again[k]) for k in got)
