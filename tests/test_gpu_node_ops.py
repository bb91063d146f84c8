"""Embedding and residual dropout against their float64 statements (``oracle.node_ops``).

Tolerances count roundings: u = eps / 2 of the output's type relative to the value for the last rounding, 2^-24 for each
float32 operation before it, half the smallest float16 step where a result is subnormal.
"""

import math

import pytest
import torch

from oracle import node_ops as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
F32 = 2.0 ** -24


def _F():
    from flashcart_amd.nn import functional as F
    return F


def _u(dtype):
    return torch.finfo(dtype).eps / 2


def _within(got, want, tol, what):
    got, want = got.detach().double().cpu(), want.double()
    assert got.shape == want.shape, what
    same = (got == want) | (got.isnan() & want.isnan())
    bad = ~same & ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, first "
                           f"{got[bad][0].item()} for {want[bad][0].item()}")


def _ids(n, rows, kind, seed):
    g = torch.Generator().manual_seed(seed)
    u = torch.rand(n, generator=g, dtype=torch.float64)
    if kind == "same":
        return torch.full((n,), rows - 1, dtype=torch.int64)
    return (u * rows if kind == "uniform" else torch.exp(u * math.log(rows + 1)) - 1).long().clamp_(0, rows - 1)


# n, rows, width: one token, odd widths, one row, few rows of many tokens, more rows than tokens, several sort passes,
# ids that fill less than a tile and more than one, runs of many pieces
EMBEDDING = [(1, 1, 1, "uniform"), (1, 300, 8, "uniform"), (5, 3, 7, "zipf"), (65, 1, 33, "same"),
             (3001, 4, 16, "uniform"), (2048, 119, 128, "zipf"), (2049, 257, 19, "uniform"), (4500, 70001, 5, "zipf"),
             (40000, 2, 3, "same"), (33000, 3000, 24, "zipf"), (20000, 60, 130, "same"), (777, 40, 2056, "zipf"),
             (70000, 17, 64, "zipf")]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,rows,width,kind", EMBEDDING)
def test_embedding(n, rows, width, kind, dtype):
    print(f"embedding n={n} rows={rows} width={width} {kind} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(n + width)
    ids = _ids(n, rows, kind, n)
    table, grad = torch.randn(rows, width, generator=gen).to(dtype), torch.randn(n, width, generator=gen).to(dtype)
    scale = 1.0 / 3.0
    t = table.to(DEV).requires_grad_(True)
    for padding in (None, int(ids[0])):
        out = _F().embedding(ids.to(DEV), t, scale, padding)
        want = O.embedding(ids, table, scale)
        _within(out, want, (_u(dtype) + 2 * F32) * want.abs() + 2.0 ** -25, "forward")
        (g,) = torch.autograd.grad(out, t, grad.to(DEV))
        want, size, count = O.embedding_grad(grad, ids, rows, scale, padding)
        # (a sum of k terms in any order: at most k roundings of partial sums that are at most the sum of sizes)
        tol = _u(dtype) * want.abs() + (count.unsqueeze(-1) + 2) * F32 * size + 2.0 ** -25 * (count.unsqueeze(-1) > 0)
        _within(g, want, tol, f"gradient, padding {padding}")
        (again,) = torch.autograd.grad(_F().embedding(ids.to(DEV), t, scale, padding), t, grad.to(DEV))
        assert torch.equal(g, again)


def test_embedding_ids_outside_and_layouts():
    """Ids outside the table, none at all, int32, of two dimensions; a strided table and gradient; a view at an odd offset."""
    F = _F()
    base = torch.randn(9, 22, device=DEV)
    table = base[:, 1::2].requires_grad_(True)  # (9, 11), strided
    ids = torch.tensor([[3, -1, 8], [9, 3, 1 << 40]], device=DEV)
    out = F.embedding(ids, table, 2.0)
    assert out.shape == (2, 3, 11)
    want = O.embedding(ids.cpu(), table.detach().cpu(), 2.0)
    _within(out, want, 0.0, "ids outside the table")
    grad = torch.randn(3, 2, 11, device=DEV).transpose(0, 1)
    (g,) = torch.autograd.grad(out, table, grad)
    _within(g, O.embedding_grad(grad.cpu(), ids.cpu(), 9, 2.0)[0], 1e-6, "gradient")
    small = torch.tensor([3, 8], dtype=torch.int32, device=DEV)
    assert torch.equal(F.embedding(small, table, 1.0, -1), table[small.long()])
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    out = F.embedding(none, table)
    assert out.shape == (0, 11)
    (g,) = torch.autograd.grad(out, table, torch.empty(0, 11, device=DEV))
    assert not g.any()
    half = torch.randn(1 + 5 * 24, device=DEV).bfloat16()[1:].view(5, 24)
    assert torch.equal(F.embedding(small.long() % 5, half), half[small.long() % 5])


def test_embedding_second_derivative():
    table = torch.randn(6, 5, device=DEV, requires_grad=True)
    ids = torch.tensor([0, 3, 3, 5, 7, 2], device=DEV)
    out = _F().embedding(ids, table, 0.5, 2)
    grad = torch.randn(6, 5, device=DEV, requires_grad=True)
    (g,) = torch.autograd.grad(out, table, grad, create_graph=True)
    cot = torch.randn(6, 5, device=DEV)
    (gg,) = torch.autograd.grad(g, grad, cot)
    want = torch.stack([0.5 * cot[i] if i in (0, 3, 5) else torch.zeros(5, device=DEV) for i in ids.tolist()])
    assert torch.equal(gg, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,rows,width", [
    (1, 63, 128), (1, 2, 4096), (130, 64, 3), (130, 65, 3), (777, 63, 130), (5000, 31, 9), (5000, 32, 9), (1536, 2, 5),
    (4096, 8, 64), (4097, 4, 16), (20011, 31, 100), (70001, 1, 1), (2500, 8, 1030)])
def test_embedding_gradient_of_few_rows(n, rows, width, dtype):
    """Small tables, around the limits of the sums that are kept per wave, with indices outside the table and the
    padding row among the others: their gradient rows, which are not finite here, add to nothing."""
    print(f"few rows n={n} rows={rows} width={width} {dtype}", flush=True)
    gen = torch.Generator().manual_seed(n + rows)
    ids, grad = _ids(n, rows, "uniform", n), torch.randn(n, width, generator=gen).to(dtype)
    padding = rows - 1 if rows > 1 else None
    dead = torch.rand(n, generator=gen) < 0.1
    ids[dead] = torch.tensor([-1, rows, 1 << 40, -(1 << 62), rows - 1 if rows > 1 else -1])[torch.arange(int(dead.sum())) % 5]
    dead = (ids < 0) | (ids >= rows) | (ids == (-1 if padding is None else padding))
    grad[dead] = float("nan")
    t = torch.randn(rows, width, generator=gen).to(dtype).to(DEV).requires_grad_(True)
    got = [torch.autograd.grad(_F().embedding(ids.to(DEV), t, 3.0, padding), t, grad.to(DEV))[0] for _ in range(2)]
    assert torch.equal(got[0], got[1])
    want, size, count = O.embedding_grad(grad[~dead], ids[~dead], rows, 3.0, None)
    tol = _u(dtype) * want.abs() + (count.unsqueeze(-1) + 2) * F32 * size + 2.0 ** -25 * (count.unsqueeze(-1) > 0)
    _within(got[0], want, tol, "gradient")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 3, 8, 1023, 4096 + 5, 300001])
@pytest.mark.parametrize("p", [0.0, 0.3, 0.9, 1.0])
def test_dropout(n, p, dtype):
    gen = torch.Generator().manual_seed(n)
    x, r, grad = (torch.randn(n, generator=gen).to(dtype) for _ in range(3))
    seed, offset = -(1 << 40) - 12345 + n, (1 << 35) + 7
    rng = torch.tensor([seed, offset], device=DEV)
    factor = 1 / (1 - p) if p < 1 else 1.0
    for res in (r, None):
        xd = x.to(DEV).requires_grad_(True)
        rd = None if res is None else res.to(DEV).requires_grad_(True)
        out = _F().dropout_add(xd, rd, p, rng)
        want = O.dropout_add(x, res, p, seed, offset)
        size = x.double().abs() * factor + (0 if res is None else res.double().abs())
        _within(out, want, _u(dtype) * want.abs() + 3 * F32 * size + 2.0 ** -25, "forward")
        grads = torch.autograd.grad(out, [xd] if rd is None else [xd, rd], grad.to(DEV))
        want = O.dropout_add(grad, None, p, seed, offset)
        _within(grads[0], want, (_u(dtype) + 2 * F32) * want.abs() + 2.0 ** -25, "gradient")
        assert rd is None or torch.equal(grads[1].cpu(), grad)


def test_dropout_drops_what_is_not_finite_and_takes_views():
    F = _F()
    rng = torch.tensor([5, 0], device=DEV)
    x = torch.full((4001,), math.nan, device=DEV)
    keep = O.dropout_keep(4001, 0.5, 5, 0)
    out = F.dropout_add(x, None, 0.5, rng).cpu()
    assert torch.equal(out.isnan(), keep) and not out[~keep].any()
    wide = torch.randn(33, 50, device=DEV).half()
    view = wide[:, 1::3]
    assert torch.equal(F.dropout_add(view, view, 0.25, rng), F.dropout_add(view.contiguous(), view.contiguous(), 0.25, rng))
    odd = torch.randn(1002, device=DEV).half()
    assert torch.equal(F.dropout_add(odd[1:], None, 0.25, rng), F.dropout_add(odd[1:].clone(), None, 0.25, rng))
    assert F.dropout_add(x[:0], None, 0.5, rng).numel() == 0


def test_dropout_past_32_bits():
    """Element numbers of more than 32 bits."""
    n = 2 ** 32 + 5
    x = torch.ones(n, dtype=torch.float16, device=DEV)
    out = _F().dropout_add(x, None, 0.5, torch.tensor([11, 3], device=DEV))
    tail = O.dropout_keep(4096 + 5, 0.5, 11, 3, first=n - 4096 - 5)
    assert torch.equal(out[-4096 - 5:].cpu() > 0, tail)
    del x, out
    torch.cuda.empty_cache()


def test_node_operators_on_a_stream_and_in_a_graph():
    """Captured on a side stream and replayed with other inputs and other random numbers, each replay against eager."""
    F = _F()
    ids = torch.randint(0, 50, (700,), device=DEV)
    table = torch.randn(50, 36, device=DEV).bfloat16().requires_grad_(True)
    rng, grad = torch.tensor([1, 2], device=DEV), torch.randn(700, 36, device=DEV).bfloat16()

    def step():
        e = F.embedding(ids, table, 6.0, 0)
        out = F.dropout_add(e, e, 0.2, rng)
        return out.detach(), torch.autograd.grad(out, table, grad)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = step()
    torch.cuda.current_stream().wait_stream(side)
    for k in range(4):
        ids.copy_(torch.randint(0, 50, (700,), device=DEV))
        rng.add_(k + 1)
        grad.normal_()
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, want)), k


def test_other_devices_and_types_are_refused():
    F = _F()
    x, rng = torch.zeros(4, 4, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    with pytest.raises(TypeError):
        F.dropout_add(x, x.half(), 0.5, rng)
    with pytest.raises(ValueError, match="differ in shape"):
        F.dropout_add(x, x[:2], 0.5, rng)
    with pytest.raises(ValueError, match="p must be"):
        F.dropout_add(x, None, 1.5, rng)
    with pytest.raises(ValueError, match="seed and an offset"):
        F.dropout_add(x, None, 0.5, rng[:1])
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        F.dropout_add(x, None, 0.5, rng.cpu())
    with pytest.raises(ValueError, match="not empty"):
        F.embedding(rng, x[:0])
