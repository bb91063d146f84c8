"""How programs use the row norm and the dense layers beyond a call at a time: more elements than 31 bits count, the same
tensor twice, other streams, captured graphs that share memory, many threads."""

import threading

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


def _small_integers(*shape, dtype=torch.bfloat16, low=-1, high=2):
    """Sums of products of them are exact in float32, and in bfloat16 as long as they stay below 256."""
    out = torch.empty(*shape, device=DEV, dtype=dtype)
    for a in range(0, shape[0], 1 << 18):
        out[a:a + (1 << 18)] = torch.randint(low, high, out[a:a + (1 << 18)].shape, device=DEV)
    return out


def test_rows_beyond_31_bits_in_a_dense_layer():
    """2^31 elements of x and of y; the weight holds one 1 in each row, so that y and dx are columns of x and of the gradient."""
    n, width, out = (1 << 21) + 5, 1032, 1040
    print(f"dense n={n} width={width} out={out}", flush=True)
    x = _small_integers(n, width, low=-100, high=101)
    pick = torch.randint(0, width, (out,), device=DEV)
    w = torch.zeros(out, width, device=DEV, dtype=torch.bfloat16)
    w[torch.arange(out, device=DEV), pick] = 1
    x.requires_grad_()
    y = _F().dense(x, w)
    for a in (0, (1 << 20) - 7, n - 300):
        assert torch.equal(y[a:a + 300], x[a:a + 300][:, pick])
    (dx,) = torch.autograd.grad(y, x, y.detach())
    for a in (0, (1 << 20) - 7, n - 300):
        want = torch.zeros(300 if a + 300 <= n else n - a, width, device=DEV)
        want.index_add_(1, pick, y[a:a + 300].detach().float())
        assert torch.equal(dx[a:a + 300], want.bfloat16())


def test_rows_beyond_31_bits_in_groups():
    n, width, out = (1 << 21) + 5, 1032, 16
    print(f"grouped n={n} width={width} out={out}", flush=True)
    x = _small_integers(n, width)
    w = _small_integers(3, out, width)
    offsets = torch.tensor([2, 1 << 20, 1 << 20, n - 1], device=DEV)
    y = _F().grouped_dense(x, w, offsets)
    assert not y[:2].any() and not y[n - 1:].any()
    for e, a, b in ((0, 2, 400), (0, (1 << 20) - 300, 1 << 20), (2, 1 << 20, (1 << 20) + 300), (2, n - 301, n - 1)):
        assert torch.equal(y[a:b], (x[a:b].float() @ w[e].float().t()).bfloat16())
    wl = w.clone().requires_grad_()
    g = torch.zeros(n, out, device=DEV, dtype=torch.bfloat16)
    g[n - 2], g[3], g[0] = 1, 2, 5
    (dw,) = torch.autograd.grad(_F().grouped_dense(x, wl, offsets), wl, g)
    assert torch.equal(dw[2], x[n - 2].expand(out, -1)) and torch.equal(dw[0], 2 * x[3].expand(out, -1)) and not dw[1].any()


def test_rows_beyond_31_bits_in_the_norm():
    n, width = (1 << 21) + 5, 1032
    x = _small_integers(n, width)
    x[:, 0] = 1
    y, total = _F().rms_norm_add(x, x)
    q, scale, _ = _F().rms_norm_add_quantized(x, x)
    for a in (0, (1 << 20) - 7, n - 300):
        t = 2 * x[a:a + 300].float()
        want = t * torch.rsqrt(t.square().mean(1, keepdim=True) + 1e-6)
        assert torch.equal(total[a:a + 300].float(), t)
        assert float((y[a:a + 300].float() - want).abs().max()) <= 2.0 ** -8 * float(want.abs().max())
        assert torch.equal(q[a:a + 300].float(), 448 * x[a:a + 300].float().sign())
        assert float((scale[a:a + 300] - want.abs().amax(1) / 448).abs().max()) <= 1e-6


def test_one_tensor_as_both_inputs():
    """x as its own residual: its gradient comes by both ways."""
    F = _F()
    x, g, gt = (torch.randn(30, 48, device=DEV) for _ in range(3))
    two = [x.clone().requires_grad_() for _ in range(2)]
    outs = F.rms_norm_add(*two)
    want = sum(torch.autograd.grad(outs, two, (g, gt)))
    one = x.clone().requires_grad_()
    (got,) = torch.autograd.grad(F.rms_norm_add(one, one), one, (g, gt))
    assert torch.equal(got, want)
    one.grad = None
    y, total = F.rms_norm_add(one, one)
    (y * g + total * gt).sum().backward()
    assert torch.equal(one.grad, want)
    w = torch.randn(48, 48, device=DEV)
    one = x.clone().requires_grad_()
    (got,) = torch.autograd.grad(F.dense(one, w, residual=one), one, g)
    assert torch.allclose(got, g + g @ w, rtol=1e-5, atol=1e-4)


def test_the_kept_total_may_not_be_changed():
    """Autograd notices that the rows which the backward pass reads were overwritten."""
    x, r = (torch.randn(4, 8, device=DEV, requires_grad=True) for _ in range(2))
    y, total = _F().rms_norm_add(x, r)
    total.detach().mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_on_another_stream():
    """The calls run on the current stream: behind a long kernel there, and not before."""
    F = _F()
    x, w = torch.randn(700, 520, device=DEV), torch.randn(300, 520, device=DEV)
    a = torch.randn(6000, 6000, device=DEV)
    want = F.dense(F.rms_norm_add(2 * x)[0], w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(3):
            a @ a
        later = x.clone().mul_(2)
        got = F.dense(F.rms_norm_add(later)[0], w)
    side.synchronize()
    assert torch.equal(got, want)


def test_two_graphs_that_share_memory():
    """Two graphs captured into one pool, replayed in turn with eager calls between: each as the eager call."""
    F = _F()
    pool = torch.cuda.graph_pool_handle()
    parts = []
    for seed, (n, width, out) in enumerate(((48, 4096, 512), (300, 700, 264))):  # (split sums; copies of operands)
        gen = torch.Generator(device=DEV).manual_seed(seed)
        t = [torch.randn(*s, device=DEV, generator=gen, dtype=torch.float32).bfloat16().requires_grad_()
             for s in ((n, width), (out, width), (out,))]
        g = torch.randn(n, out, device=DEV, generator=gen).bfloat16()
        parts.append((t, g))

    def step(part):
        t, g = part
        y = F.dense(*t, "silu", 1.0, t[0].shape[1] ** -0.5)
        return (y.detach(), *torch.autograd.grad(y, t, g))

    graphs, held = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for part in parts:
            step(part)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side, pool=pool):
                held.append(step(part))
            graphs.append(graph)
    torch.cuda.current_stream().wait_stream(side)
    for turn in range(4):
        for k in (0, 1) if turn % 2 else (1, 0):
            with torch.no_grad():
                parts[k][0][0].normal_()
            graphs[k].replay()
            torch.cuda.synchronize()
            seen = [t.clone() for t in held[k]]
            assert all(torch.equal(a, b) for a, b in zip(seen, step(parts[k]))), (turn, k)


def test_from_several_threads():
    """Threads with streams of their own, each with sizes of its own: as one after the other."""
    F = _F()
    sizes = [(5, 300, 77), (130, 264, 1032), (64, 2048, 512), (1000, 96, 40)]
    inputs = [(torch.randn(n, a, device=DEV), torch.randn(b, a, device=DEV)) for n, a, b in sizes]
    want = [F.dense(x, w, act="gelu", scale=0.1) for x, w in inputs]
    torch.cuda.synchronize()
    got = [None] * len(sizes)

    def work(k):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                got[k] = F.dense(*inputs[k], act="gelu", scale=0.1)
            torch.cuda.current_stream().synchronize()

    threads = [threading.Thread(target=work, args=(k,)) for k in range(len(sizes))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
