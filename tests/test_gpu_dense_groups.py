"""Dense layers of very many groups, whose units stand in a table: as the same rows call by call, and offsets of any value."""

import pytest
import torch

from oracle import node_ops as O
from tests.test_gpu_dense import DEV, DTYPES, _F, _check, _inputs, _roundings, _run

pytestmark = pytest.mark.gpu


def _offsets(groups, n, kind, seed):
    gen = torch.Generator().manual_seed(seed)
    if kind == "even":
        return torch.arange(groups + 1) * n // groups
    if kind == "uneven":  # most groups are empty, some have many rows; rows in none at both ends
        ends = torch.randint(5, n - 9, (groups // 8,), generator=gen).sort().values
        return torch.cat([torch.tensor([5]), ends.repeat_interleave(8), torch.full((groups - groups // 8 * 8,), n - 9)])
    off = torch.randint(-3 * n, 4 * n, (groups + 1,), generator=gen)  # anything
    off[::3] = torch.arange(0, groups + 1, 3) * n // groups
    off[7] = -2 ** 62
    return off


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["even", "uneven", "any"])
@pytest.mark.parametrize("groups,n,width,out", [(257, 900, 40, 24), (1025, 5000, 33, 70), (5000, 3000, 17, 9), (300, 30000, 128, 136),
                                                (65536, 4000, 8, 8)])
def test_many_groups(groups, n, width, out, kind, dtype):
    print(f"groups={groups} n={n} width={width} out={out} {kind} {dtype}", flush=True)
    x, w, b, _, grad = _inputs(n, width, out, dtype, groups=groups, seed=31)
    off = _offsets(groups, n, kind, groups).to(DEV)
    args = ("silu", 1.6, width ** -0.5)
    got = _run(x, w, b, None, *args, grad, off)
    ends = torch.cummax(off.clamp(0, n), 0).values
    rows = torch.arange(n, device=DEV)
    at = torch.searchsorted(ends, rows, right=True) - 1
    inside = (at >= 0) & (at < groups)
    assert not got["y"][~inside].any() and not got["dx"][~inside].any()
    if not inside.any():
        return
    # the rows of a group are one layer: y and dx row by row, dw and db as sums over the rows of each
    f = 2.0 ** -24
    e, X, W, B, G = at[inside], x[inside].double(), w.double(), b.double(), grad[inside].double()
    z = args[2] * torch.bmm(W[e], X[:, :, None])[:, :, 0] + B[e]
    e_z = (width + 4) * f * (args[2] * torch.bmm(W[e].abs(), X.abs()[:, :, None])[:, :, 0] + z.abs())
    a, d = O.activation(z, "silu")
    r = _roundings(dtype)
    e_a, e_d = 1.13 * e_z + 16 * f * (1 + z.abs()), 0.8 * e_z + 16 * f * (1 + z.abs())
    want = {"y": (1.6 * a, r["end"] * 1.6 * a.abs() + 1.6 * (e_a + 2 * f * a.abs()) + r["tiny"])}
    dz = 1.6 * G * d
    m_dz = (1.6 * G).abs() * (e_d + (r["kept"] + 3 * f) * d.abs()) + r["mid"] * dz.abs() + r["tiny"]
    s = args[2]
    dx = s * torch.bmm(dz[:, None], W[e])[:, 0]
    want["dx"] = (dx, r["end"] * dx.abs() + s * torch.bmm((m_dz + (out + 3) * f * dz.abs())[:, None], W[e].abs())[:, 0] + r["tiny"])
    zero = torch.zeros(groups, out, width, device=DEV, dtype=torch.float64)

    def sums(u, v):
        return zero.index_add(0, e, u[:, :, None] * v[:, None, :])

    most = int(torch.bincount(e).max())
    dw = s * sums(dz, X)
    want["dw"] = (dw, r["end"] * dw.abs() + s * sums(m_dz + (most + 3) * f * dz.abs(), X.abs()) + r["tiny"])
    flat = torch.zeros(groups, out, device=DEV, dtype=torch.float64)
    db = flat.index_add(0, e, dz)
    size = flat.index_add(0, e, (1.6 * G).abs() * (e_d + (r["kept"] + 3 * f) * d.abs()) + (most + 3) * f * dz.abs())
    want["db"] = (db, r["end"] * db.abs() + size + r["tiny"])
    _check({"y": got["y"][inside], "dx": got["dx"][inside], "dw": got["dw"], "db": got["db"]}, want, dtype)
    again = _run(x, w, b, None, *args, grad, off)
    assert all(torch.equal(got[k], again[k]) for k in got)


def test_many_groups_in_a_graph():
    """The table is made again at every replay, from the offsets as they are then."""
    x, w, b, _, grad = _inputs(2000, 48, 40, torch.bfloat16, groups=700, seed=32)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    off = _offsets(700, 2000, "even", 0).to(DEV)

    def step():
        y = _F().grouped_dense(*leaves[:2], off, leaves[2], "gelu", 1.0, 0.15)
        return (y.detach(), *torch.autograd.grad(y, leaves, grad))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.current_stream().wait_stream(side)
    for k, kind in enumerate(("uneven", "any", "even", "any")):
        off.copy_(_offsets(700, 2000, kind, k))
        graph.replay()
        torch.cuda.synchronize()
        seen = [t.clone() for t in held]
        assert all(torch.equal(a, c) for a, c in zip(seen, step())), kind
