"""Dense layers of more workgroups than one launch has: very many groups or rows. Values are -1, 0 and 1, whose sums are exact."""

import pytest
import torch

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


def _small_integers(*shape, seed=0):
    out = torch.empty(*shape, device=DEV, dtype=torch.bfloat16)
    gen = torch.Generator(device=DEV).manual_seed(seed)
    flat = out.view(-1)
    for a in range(0, flat.numel(), 1 << 28):
        part = flat[a:a + (1 << 28)]
        part.copy_(torch.randint(-1, 2, part.shape, device=DEV, generator=gen, dtype=torch.int8))
    return out


# 2^24 workgroups of the kernel for few rows, of the bias' gradient 2^23; 2^20 and more of tiles, whatever their size
@pytest.mark.parametrize("groups,width,out,n", [(16384, 1, 16384, 20), (2100, 8, 1 << 17, 300)])
def test_many_groups(groups, width, out, n):
    print(f"groups={groups} width={width} out={out} n={n}", flush=True)
    x, w, b, g = (_small_integers(*s, seed=k).requires_grad_(k < 3)
                  for k, s in enumerate(((n, width), (groups, out, width), (groups, out), (n, out))))
    at = torch.randint(0, groups, (n,), generator=torch.Generator().manual_seed(1)).sort().values.to(DEV)
    at[:2], at[-2:] = 0, groups - 1
    offsets = torch.searchsorted(at, torch.arange(groups + 1, device=DEV))
    y = _F().grouped_dense(x, w, offsets, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    with torch.no_grad():
        want = torch.bmm(w[at].float(), x.float()[:, :, None])[:, :, 0] + b[at].float()
        assert torch.equal(y, want.bfloat16())
        assert torch.equal(dx, torch.bmm(g.float()[:, None], w[at].float())[:, 0].bfloat16())
        used = at.unique()
        for e in used.tolist():
            rows = at == e
            assert torch.equal(dw[e], (g[rows].float().t() @ x[rows].float()).bfloat16()), e
            assert torch.equal(db[e], g[rows].float().sum(0).bfloat16()), e
        empty = torch.ones(groups, dtype=torch.bool, device=DEV)
        empty[used] = False
        for e in range(0, groups, 512):
            part = slice(e, e + 512)
            assert not dw[part][empty[part]].any() and not db[part][empty[part]].any()


def test_many_rows():
    n, width, out = (1 << 26) + 77, 8, 8
    x, w, b, g = (_small_integers(*s, seed=k).requires_grad_(k < 3)
                  for k, s in enumerate(((n, width), (out, width), (out,), (n, out))))
    y = _F().dense(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), g)
    sums, bias = torch.zeros(out, width, dtype=torch.float64, device=DEV), torch.zeros(out, dtype=torch.float64, device=DEV)
    with torch.no_grad():
        for a in range(0, n, 1 << 23):
            part = slice(a, a + (1 << 23))
            xf, gf = x[part].float(), g[part].float()
            assert torch.equal(y[part], (xf @ w.float().t() + b.float()).bfloat16()), a
            assert torch.equal(dx[part], (gf @ w.float()).bfloat16()), a
            sums += gf.double().t() @ xf.double()
            bias += gf.double().sum(0)
    assert torch.equal(dw, sums.bfloat16()) and torch.equal(db, bias.bfloat16())


@pytest.mark.parametrize("offsets", [None, [0, 1 << 20, 1 << 20, (1 << 20) + 40, 1 << 22]])
@pytest.mark.parametrize("alone", [False, True])
def test_bias_gradient_of_many_rows(offsets, alone):
    """A float32 sum of n equal numbers whose additions are no longer chain than 4 + 8 + 64 + 512 + 32 is off by at most
    2^-24 of it for each. (Other numbers in the last rows, so that a part taken twice or left out shows.)"""
    n, out = 1 << 22, 8
    g = torch.full((n, out), 0.1, device=DEV)
    g[-5000:] = torch.arange(out, device=DEV) + 1.0
    g[(1 << 20) - 70:1 << 20] = 3.0
    x = torch.ones(n, 8, device=DEV, requires_grad=not alone)
    w = torch.ones(*(() if offsets is None else (4,)), out, 8, device=DEV)
    b = torch.zeros(w.shape[:-1], device=DEV, requires_grad=True)
    y = _F().dense(x, w, b) if offsets is None else _F().grouped_dense(x, w, torch.tensor(offsets, device=DEV), b)
    db = torch.autograd.grad(y, b if alone else (b, x), g)[0]
    if offsets is None:
        want = g.double().sum(0)
    else:
        want = torch.stack([g[p:q].double().sum(0) for p, q in zip(offsets, offsets[1:])])
    off = (db.double() - want).abs()
    assert bool((off <= 620 * 2.0 ** -24 * want).all()), float((off / want.clamp_min(1e-30)).max())


@pytest.mark.parametrize("groups", [3, 1000])
def test_bias_gradients_of_many_rows_in_groups(groups):
    """Uneven groups, each sum exact: more than one level of sums, in groups of none, one and many of their parts."""
    n, out = (1 << 21) + 333, 264
    gen = torch.Generator().manual_seed(groups)
    ends = torch.randint(0, n + 1, (groups - 1,), generator=gen).sort().values
    offsets = torch.cat([torch.tensor([5]), ends.clamp(min=5), torch.tensor([n - 9])]).clamp(max=n - 9).to(DEV)
    x = torch.zeros(n, 8, device=DEV)
    b = torch.zeros(groups, out, device=DEV, requires_grad=True)
    g = _small_integers(n, out).float()
    (db,) = torch.autograd.grad(_F().grouped_dense(x, torch.zeros(groups, out, 8, device=DEV), offsets, b), b, g)
    sums = torch.cat([torch.zeros(1, out, device=DEV, dtype=torch.float64), g.double().cumsum(0)])
    assert torch.equal(db.double(), sums[offsets[1:]] - sums[offsets[:-1]])
