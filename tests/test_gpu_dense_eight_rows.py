"""8-bit dense layers of few rows on both sides of the rule between their two kernels, against float64 products of the same 8-bit
numbers."""

import ctypes

import pytest
import torch

from oracle import node_ops as O
from tests.test_gpu_dense import DEV, _F, _inputs, _roundings

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,width,out,few", [(1, 4096, 4096, True), (16, 8192, 1032, True), (17, 4096, 4096, True), (32, 4112, 512, False),
                                             (32, 512, 4112, False), (33, 64, 64, False), (16, 4097, 4096, True), (5, 8195, 515, True),
                                             (3, 4097, 10240, False), (32, 2055, 4091, True), (32, 4097, 4099, False)])
def test_few_rows(n, width, out, few):
    from flashcart_amd import _lib
    print(f"8 bits n={n} width={width} out={out}", flush=True)
    # (rows that are not whole chunks are copied for tiles, and asked for as such: aligned or not is the same to them)
    desc = _lib.DenseDesc(1, 0, width, out, 0, 1, 1.0, 1.0)
    assert (_lib.load().fc_node_dense_tile(desc, n, 1, ctypes.byref(ctypes.c_int32())) == 0) == few
    x, w, b, res, _ = _inputs(n, width, out, torch.bfloat16, seed=30)
    (qx, sx), (qw, sw) = _F().quantize_rows(x), _F().quantize_rows(w)
    xv, wv = qx.double() * sx.double()[:, None], qw.double() * sw.double()[:, None]
    scale = width ** -0.5
    y, bound = O.dense(xv, wv, b, res, "silu", 1.6, scale, **_roundings(torch.bfloat16))["y"]
    got = _F().quantized_dense(qx, sx, qw, sw, b, "silu", 1.6, scale, res)
    # the instruction may lose 2^-13 of the largest of its 8 products in each
    most = (xv.abs().amax(1)[:, None] * wv.abs().amax(1)) * width * 2.0 ** -13 * scale * 1.6 * 1.13
    assert bool(((got.double() - y).abs() <= bound + most).all())
    assert float((got.double() - y).norm()) <= 0.9 * torch.finfo(torch.bfloat16).eps / 2 * float(y.norm()) or y.numel() < 1000
