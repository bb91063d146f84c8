"""Node-wise operators on more elements than 31 and 32 bits count, and on more 16-byte chunks than a grid has threads
(2^32). Tensors are up to 64 GiB; what is compared is all of the cheap ones, and the beginning, the end and the borders of
launches of the others."""

import math

import pytest
import torch

from oracle import node_ops as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _F():
    from flashcart_amd.nn import functional as F
    return F


@pytest.fixture(autouse=True)
def _memory_is_given_back():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def test_dropout_of_more_chunks_than_threads():
    n = 2 ** 35 + 4101
    print(f"dropout n={n} float16", flush=True)
    x = torch.ones(n, dtype=torch.float16, device=DEV)
    out = _F().dropout_add(x, None, 0.5, torch.tensor([11, 3], device=DEV))
    del x
    # (2^31: elements of one launch)
    for first in (0, 2 ** 31 - 512, 2 ** 32 - 512, 2 ** 35 - 2 ** 31 - 512, 2 ** 35 - 512, n - 1021):
        part = out[first:first + 1021].cpu()
        assert torch.equal(part, 2.0 * O.dropout_keep(part.numel(), 0.5, 11, 3, first=first).half()), first


@pytest.mark.parametrize("n,width,dtype", [(2 ** 25 + 3, 1024, torch.float16), (2 ** 21 + 3, 1030, torch.float32),
                                           (3, 2 ** 31 - 65536, torch.bfloat16)])
def test_embedding_lookup(n, width, dtype):
    print(f"lookup n={n} width={width} {dtype}", flush=True)
    table = torch.randn(2 if width > 10 ** 6 else 5, width, device=DEV, dtype=dtype)
    ids = torch.randint(0, table.shape[0], (n,), device=DEV)
    out = _F().embedding(ids, table)
    step = max(1, (1 << 30) // width)
    for a in range(0, n, step):
        assert torch.equal(out[a:a + step], table[ids[a:a + step]]), a


def _small_integers(n, width, dtype):
    """-1, 0 and 1: sums of fewer than 2^24 of them are exact in float32 in any order."""
    out = torch.empty(n, width, device=DEV, dtype=dtype)
    for a in range(0, n, 1 << 18):
        out[a:a + (1 << 18)] = torch.randint(-1, 2, out[a:a + (1 << 18)].shape, device=DEV)
    return out


@pytest.mark.parametrize("n,rows,width", [(2 ** 21 + 5, 40000, 1030), (2 ** 21 + 5, 6, 1030), (700, 2 ** 21 + 9, 1030)])
def test_embedding_gradient(n, rows, width):
    """Long gradients, sorted and summed per wave, and a long table: every element, exactly."""
    print(f"gradient n={n} rows={rows} width={width}", flush=True)
    grad = _small_integers(n, width, torch.float16)
    ids = torch.randint(0, rows, (n,), device=DEV)
    ids[-1] = rows - 1
    got = torch.ops.flashcart.embedding_bwd(grad, ids, rows, 1.0, 1)
    if rows < n:
        want = torch.zeros(rows, width, device=DEV)
        for a in range(0, n, 1 << 18):
            want.index_add_(0, ids[a:a + (1 << 18)], grad[a:a + (1 << 18)].float())
        want[1] = 0
        assert torch.equal(got, want.half())
        return
    used = ids.unique()
    want = torch.zeros(used.numel(), width, device=DEV).index_add_(0, torch.searchsorted(used, ids), grad.float())
    want[used == 1] = 0
    assert torch.equal(got[used], want.half())
    got[used] = 0
    assert all(not part.any() for part in got.split(1 << 18))


# the padded copy of x takes more than one launch; more than 2^31 hidden values; x and y in float32
@pytest.mark.parametrize("n,width,hidden,dtype", [(2 ** 24 + 3, 129, 8, torch.float16), (2 ** 21 + 7, 8, 1032, torch.bfloat16),
                                                  (2 ** 24 + 3, 130, 8, torch.float32)])
def test_feed_forward(n, width, hidden, dtype):
    """Rows at both ends and in the middle, and the weights' gradients of these rows (those of the others get none)."""
    from tests.test_gpu_feed_forward import NAMES, _roundings
    print(f"feed-forward n={n} width={width} hidden={hidden} {dtype}", flush=True)
    gen = torch.Generator(device=DEV).manual_seed(7)
    w_in, w_out = (torch.randn(*s, device=DEV, generator=gen).to(dtype) for s in ((2 * hidden, width), (width, hidden)))
    x = torch.empty(n, width, device=DEV, dtype=dtype)
    for part in x.split(1 << 21):
        part.normal_(generator=gen)
    spans = [(0, 300), (n // 2, n // 2 + 300), (n - 300, n)]
    rows = torch.cat([torch.arange(a, b, device=DEV) for a, b in spans])
    grad = torch.zeros_like(x)
    grad[rows] = torch.randn(rows.numel(), width, device=DEV, generator=gen).to(dtype)
    args = ("silu", 1.0, width ** -0.5, hidden ** -0.5)
    want = O.gated_feed_forward(x[rows], w_in, w_out, *args, grad[rows], **_roundings(dtype))
    leaves = [t.requires_grad_(True) for t in (x, w_in, w_out)]
    y = _F().gated_feed_forward(*leaves, *args)
    dx, dwi, dwo = torch.autograd.grad(y, leaves, grad)
    for name, got in zip(NAMES, (y.detach()[rows], dx[rows], dwi, dwo)):
        ref, bound = want[name]
        off = (got.double() - ref).abs()
        assert bool((off <= bound).all()), f"{name}: {float((off / bound).max())} times the bound"
    assert math.isclose(float(dx.abs().max()), float(dx[rows].abs().max()))  # (a row without a gradient has none)
