"""What the library says about the tiles of a dense layer, without a GPU (it then counts with 256 CUs)."""

import ctypes

import pytest


def _tile(n, which, **desc):
    from flashcart_amd import _lib
    d = dict(dtype=1, act=0, in_=2056, out=4872, groups=0, aligned=1, act_scale=1.0, scale=1.0)
    return _lib.load().fc_node_dense_tile(_lib.DenseDesc(**{**d, **desc}), n, which, None)


def test_tiles_by_size():
    halves = ctypes.c_int32(-1)
    from flashcart_amd import _lib
    desc = _lib.DenseDesc(1, 0, 64, 64, 0, 1, 1.0, 1.0)
    assert _lib.load().fc_node_dense_tile(desc, 1, 0, halves) == 0 and halves.value == 0  # the kernel for few rows
    assert _tile(4360, 0) == 256 and _tile(64, 0, groups=64, in_=2048, out=1024) == 32
    assert _tile(4360, 2) == 256 and _tile(100, 2, in_=64, out=64) == 64 and _tile(4360, 1, in_=4112) == 256


@pytest.mark.parametrize("n,which,desc,status", [
    (0, 0, {}, 4), (-1, 0, {}, 4), (1 << 27, 0, {}, 4), (8, 3, {}, 1), (8, -1, {}, 1), (8, 0, {"dtype": 3}, 1), (8, 2, {"in_": 0}, 4),
    (8, 1, {"dtype": 0}, 1), (8, 1, {"groups": 2}, 1)])
def test_bad_questions(n, which, desc, status):
    assert _tile(n, which, **desc) == -status


def test_null():
    from flashcart_amd import _lib
    assert _lib.load().fc_node_dense_tile(None, 8, 0, None) == -5
