"""The row norm and the dense layers without a GPU: refusals, shapes of fake tensors, what the autograd formulas do around
their kernels, status codes of the C entry points."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

from flashcart_amd.nn import functional as F
from oracle import node_ops as O

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
F8 = torch.float8_e4m3fn


def _eight(*shape):
    return torch.empty(*shape, dtype=F8)


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 4), torch.zeros(3, 4)
    for call in (lambda: F.rms_norm_add(x), lambda: F.rms_norm_add(x, x, w[0]), lambda: F.rms_norm_add_quantized(x),
                 lambda: F.quantize_rows(x), lambda: F.dense(x, w, w[:, 0], "silu", residual=x[:, :3]),
                 lambda: F.grouped_dense(x, w[None], torch.tensor([0, 2])),
                 lambda: F.quantized_dense(x.to(F8), x[:, 0], w.to(F8), w[:, 0])):
        with pytest.raises(RuntimeError, match="ROCm devices only"):
            call()


@pytest.mark.parametrize("call,error", [
    (lambda: F.rms_norm_add(torch.zeros(2, 4, dtype=torch.float64)), "float32, bfloat16"),
    (lambda: F.rms_norm_add_quantized(torch.zeros(2, 4, dtype=torch.int32)), "float32, bfloat16"),
    (lambda: F.dense(torch.zeros(2, 4), torch.zeros(3, 4), act="tanh"), "act must be None or one of"),
    (lambda: F.dense(torch.zeros(2, 4, dtype=torch.float64), torch.zeros(3, 4)), "float32, bfloat16"),
    (lambda: F.dense(torch.zeros(2, 4), torch.zeros(3)), "weight must be"),
    (lambda: F.dense(torch.zeros(2, 4), torch.zeros(3, 5)), "do not match"),
    (lambda: F.dense(torch.zeros(2, 4), torch.zeros(0, 4)), "not empty"),
    (lambda: F.grouped_dense(torch.zeros(2, 4), torch.zeros(1, 3, 4), None), "must be a tensor"),
    (lambda: F.grouped_dense(torch.zeros(2, 4), torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64)), "weight must be"),
    (lambda: F.grouped_dense(torch.zeros(1, 2, 4), torch.zeros(1, 3, 4), torch.zeros(2, dtype=torch.int64)), "do not match"),
    (lambda: F.quantized_dense(torch.zeros(2, 4), torch.zeros(2), _eight(3, 4), torch.zeros(3), dtype=torch.float32), "dtype"),
])
def test_arguments_are_refused(call, error):
    with pytest.raises((TypeError, ValueError), match=error):
        call()


@pytest.mark.parametrize("name", ["rms_norm_add_quantized", "quantize_rows", "quantized_dense"])
def test_gradients_through_eight_bits_are_refused(name):
    x, b = torch.zeros(2, 4), torch.zeros(3, dtype=torch.bfloat16)
    call = {"rms_norm_add_quantized": lambda t, b: F.rms_norm_add_quantized(t), "quantize_rows": lambda t, b: F.quantize_rows(t),
            "quantized_dense": lambda t, b: F.quantized_dense(t.to(F8), t[:, 0], _eight(3, 4), torch.zeros(3), b)}[name]
    with pytest.raises(NotImplementedError, match="no derivatives"):
        call(x.clone().requires_grad_(), b.clone().requires_grad_())
    with torch.no_grad(), pytest.raises(RuntimeError, match="ROCm devices only"):  # (goes on to the kernel)
        call(x.clone().requires_grad_(), b.clone().requires_grad_())
    with forward_ad.dual_level(), torch.no_grad(), pytest.raises(NotImplementedError, match="no derivatives"):
        dual = forward_ad.make_dual(x, x)
        call(dual, forward_ad.make_dual(b, b) if name == "quantized_dense" else b)


def test_fake_tensors_have_the_shapes():
    with FakeTensorMode():
        x, r, w = torch.empty(2, 5, 6, dtype=torch.float16), torch.empty(2, 5, 6, dtype=torch.float16), torch.empty(6, dtype=torch.float16)
        y, total = F.rms_norm_add(x, r, w)
        assert y.shape == total.shape == (2, 5, 6) and total is not x and F.rms_norm_add(x)[1] is x
        q, scale, total = F.rms_norm_add_quantized(x, r, w)
        assert q.shape == total.shape == x.shape and q.dtype == F8 and scale.shape == (2, 5) and scale.dtype == torch.float32
        weight, bias = torch.empty(7, 6, dtype=torch.float16), torch.empty(7, dtype=torch.float16)
        y = F.dense(x, weight, bias, "gelu", residual=torch.empty(2, 5, 7, dtype=torch.float16))
        assert y.shape == (2, 5, 7) and y.dtype == torch.float16
        y = F.grouped_dense(x[0], weight[None], torch.empty(2, dtype=torch.int32), bias[None])
        assert y.shape == (5, 7)
        y = F.quantized_dense(q, scale, *F.quantize_rows(weight), bias, dtype=torch.float16)
        assert y.shape == (2, 5, 7) and y.dtype == torch.float16


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", [0, 3])
@pytest.mark.parametrize("n,width,out", [(1, 1, 1), (7, 24, 41), (600, 520, 523), (2000, 1024, 1024), (0, 8, 8)])
def test_kept_bytes_of_fake_tensors(n, width, out, act, dtype):
    """The shape-only operator keeps as many bytes as the library asks for."""
    from flashcart_amd import _lib
    want = _lib.load().fc_node_dense_saved(_lib.DenseDesc(DTYPES.index(dtype), act, width, out, 0, 1, 1.0, 1.0), n)
    with FakeTensorMode():
        x, w = torch.empty(n, width, dtype=dtype), torch.empty(out, width, dtype=dtype)
        saved = torch.ops.flashcart.node_dense(x, w, None, None, None, act, 1.0, 1.0, True)[1]
    assert saved.numel() == want


def _calls():
    """Operators as functions of one differentiable argument, that argument, and the operator of the backward pass."""
    x, r, w = torch.empty(5, 4), torch.empty(5, 4), torch.empty(4)
    weight, bias, res = torch.empty(6, 4), torch.empty(6), torch.empty(5, 6)
    off = torch.zeros(3, dtype=torch.int64)
    group = torch.empty(2, 6, 4)
    norm, lin = "flashcart::rms_norm_add_bwd", "flashcart::node_dense_bwd"
    return {
        "norm x": (lambda t: F.rms_norm_add(t, r, w)[0], x, norm),
        "norm without residual": (lambda t: F.rms_norm_add(t, None, w)[0], x, norm),
        "norm residual": (lambda t: F.rms_norm_add(x, t, w)[0], r, norm),
        "norm weight": (lambda t: F.rms_norm_add(x, r, t)[0], w, norm),
        "norm weight alone": (lambda t: F.rms_norm_add(x, None, t)[0], w, norm),
        "norm total": (lambda t: F.rms_norm_add(x, t, w)[1], r, None),
        "dense x": (lambda t: F.dense(t, weight, bias, "silu", residual=res), x, lin),
        "dense weight": (lambda t: F.dense(x, t), weight, lin),
        "dense bias": (lambda t: F.dense(x, weight, t), bias, lin),
        "dense residual": (lambda t: F.dense(x, weight, None, "silu", residual=t), res, None),
        "dense residual beside a bias": (lambda t: F.dense(x, weight, bias, "silu", residual=t), res, None),
        "grouped x": (lambda t: F.grouped_dense(t, group, off), x, lin),
        "grouped weight": (lambda t: F.grouped_dense(x, t, off, torch.empty(2, 6)), group, lin),
        "grouped bias": (lambda t: F.grouped_dense(x, group, off, t), torch.empty(2, 6), lin),
    }


NAMES = list(_calls())


class _Calls(TorchDispatchMode):
    """The operators that run, without queries of properties and views (a kept output is unpacked as one)."""

    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace != "prim" and func.name() != "aten::detach":
            self.names.append(func.name())
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("name", NAMES)
def test_backward_passes_run_their_operator_alone(name):
    """One operator, or none where the gradient is passed on; no zeros for outputs without a gradient."""
    with FakeTensorMode():
        call, t, op = _calls()[name]
        out = call(t.requires_grad_())
        grad = torch.empty_like(out)
        with _Calls() as calls:
            (got,) = torch.autograd.grad(out, t, grad)
    assert got.shape == t.shape and calls.names == ([] if op is None else [op])


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("enabled", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_forward_mode_is_refused(name, enabled, recorded):
    """A tangent is never dropped: forward-mode derivatives, which the operators lack, raise."""
    with FakeTensorMode(), forward_ad.dual_level(), torch.set_grad_enabled(enabled):
        call, t, _ = _calls()[name]
        dual = forward_ad.make_dual(t.requires_grad_(recorded), torch.empty_like(t))
        with pytest.raises(RuntimeError, match="jvp is not implemented"):
            call(dual)
        assert call(t).requires_grad == (enabled and recorded)  # (the level alone refuses nothing)


def test_both_outputs_of_the_norm():
    """Gradients of y and of the total go through one call; either may be missing."""
    with FakeTensorMode():
        x, r, w = (torch.empty(*s).requires_grad_() for s in ((5, 4), (5, 4), (4,)))
        y, total = F.rms_norm_add(x, r, w)
        g = torch.empty(5, 4)
        with _Calls() as calls:
            grads = torch.autograd.grad((y, total), (x, r, w), (g, g))
        assert calls.names == ["flashcart::rms_norm_add_bwd"] and [t.shape for t in grads] == [(5, 4), (5, 4), (4,)]


def test_library_refuses_bad_arguments():
    """Status codes of the C entry points, decided before anything is launched."""
    from flashcart_amd import _lib
    lib = _lib.load()
    bad_desc, shape, null, workspace = 1, 4, 5, 6
    # the norm
    assert lib.fc_row_norm_fwd(3, 1, 8, 16, None, None, 1e-6, None, 16, None, None) == bad_desc
    for n, width in ((-1, 8), (1, 0), (1, (1 << 20) + 1), (1 << 31, 8)):
        assert lib.fc_row_norm_fwd(0, n, width, 16, None, None, 1e-6, None, 16, None, None) == shape
        assert lib.fc_row_norm_bwd_workspace(0, n, width, 1) == -shape
    assert lib.fc_row_norm_fwd(0, 1, 8, None, None, None, 1e-6, None, 16, None, None) == null
    assert lib.fc_row_norm_fwd(0, 1, 8, 16, 16, None, 1e-6, None, 16, None, None) == null  # no total
    assert lib.fc_row_norm_fwd(0, 0, 8, None, None, None, 1e-6, None, None, None, None) == 0
    assert lib.fc_row_norm_quantize(0, 0, 1, 8, 16, 16, None, 0.0, 16, 16, 16, None) == bad_desc
    assert lib.fc_row_norm_quantize(0, 1, 1, 8, 16, None, None, 0.0, None, 16, None, None) == null
    need = lib.fc_row_norm_bwd_workspace(1, 100, 16, 1)
    assert need > 0 and lib.fc_row_norm_bwd_workspace(1, 100, 16, 0) == 0
    assert lib.fc_row_norm_bwd(1, 100, 16, 16, None, 16, None, 16, 16, 16, 16, need - 1, None) == workspace
    assert lib.fc_row_norm_bwd(1, 100, 16, 16, None, 16, None, 16, 16, 16, 18, need, None) == workspace
    assert lib.fc_row_norm_bwd(1, 100, 16, 16, None, 16, None, None, 16, None, None, 0, None) == null
    assert lib.fc_row_norm_bwd(1, 0, 16, 16, None, 16, None, 16, None, 16, 16, 64, None) == shape
    # dense layers
    good = dict(dtype=1, act=0, in_=8, out=16, groups=0, aligned=0, act_scale=1.0, scale=1.0)
    d = _lib.DenseDesc(**good)
    size = lib.fc_node_dense_fwd_workspace(d, 3)
    assert size >= 0 and lib.fc_node_dense_saved(d, 3) == 3 * 16 * 2 and lib.fc_node_dense_saved(d, -1) == -shape
    assert lib.fc_node_dense_fwd(d, 3, 16, None, None, None, None, 16, None, 16, size, None) == null
    big = lib.fc_node_dense_fwd_workspace(d, 1000)  # (operands are copied)
    assert big > 0 and lib.fc_node_dense_fwd(d, 1000, 16, 16, None, None, None, 16, None, 16, big - 1, None) == workspace
    assert lib.fc_node_dense_fwd(d, 1000, 16, 16, None, None, None, 16, 18, 16, big, None) == workspace
    bwd = lib.fc_node_dense_bwd_workspace(d, 3, 1, 1, 1)
    assert bwd > 0
    assert lib.fc_node_dense_bwd(d, 3, 16, 16, 16, 16, None, 16, 16, 16, 16, bwd - 1, None) == workspace
    assert lib.fc_node_dense_bwd(d, 3, 16, 16, 16, None, None, 16, 16, 16, 16, bwd, None) == null  # nothing kept
    assert lib.fc_node_dense_bwd(d, 0, 16, 16, 16, 16, None, None, 16, None, 16, bwd, None) == shape
    assert lib.fc_node_dense_bwd(d, 3, 16, 16, 16, 16, None, None, None, None, None, 0, None) == 0  # nothing asked for
    d = _lib.DenseDesc(**{**good, "aligned": 1})
    assert lib.fc_node_dense_fwd(d, 3, 18, 16, None, None, None, 16, None, 16, 1 << 20, None) == bad_desc
    d = _lib.DenseDesc(**{**good, "groups": 2})
    assert lib.fc_node_dense_fwd(d, 3, 16, 16, None, None, None, 16, None, 16, 1 << 20, None) == null  # no offsets
    assert lib.fc_node_dense_fwd(d, 3, 16, 16, None, 16, 16, 16, None, 16, 1 << 20, None) == bad_desc  # a residual
    for bad, code in ((dict(dtype=3), bad_desc), (dict(act=4), bad_desc), (dict(in_=0), shape),
                      (dict(out=(1 << 20) + 1), shape), (dict(groups=-1), shape), (dict(groups=(1 << 16) + 1), shape),
                      (dict(groups=1 << 16, out=1 << 15), shape)):
        d = _lib.DenseDesc(**{**good, **bad})
        assert lib.fc_node_dense_saved(d, 3) == -code and lib.fc_node_dense_fwd_workspace(d, 3) == -code
        assert lib.fc_node_dense_bwd_workspace(d, 3, 1, 1, 1) == -code
    assert lib.fc_quantized_dense_workspace(_lib.DenseDesc(**{**good, "dtype": 0}), 3) == -bad_desc
    assert lib.fc_quantized_dense_workspace(_lib.DenseDesc(**{**good, "groups": 1}), 3) == -bad_desc
    assert lib.fc_quantized_dense(_lib.DenseDesc(**good), 3, 16, None, 16, 16, None, None, 16, 16, 1 << 20, None) == null


def test_compilers_see_the_operators():
    """One graph with the operators themselves in it (which then end in their own error on the CPU)."""
    seen = []

    def backend(graph, inputs):
        seen.extend(str(n.target) for n in graph.graph.nodes if n.op == "call_function")
        return graph.forward

    def block(x, weight, group, offsets):
        y, total = F.rms_norm_add(x, x, weight[0])
        return F.dense(F.grouped_dense(y, group, offsets), weight, act="silu", residual=total)

    with pytest.raises(RuntimeError, match="ROCm devices only"):
        torch.compile(block, backend=backend, fullgraph=True)(torch.zeros(2, 4), torch.zeros(4, 4), torch.zeros(1, 4, 4),
                                                              torch.tensor([0, 2]))
    for name in ("rms_norm_add", "node_dense"):
        assert any(f"flashcart.{name}.default" in t for t in seen)


def test_oracle_against_torch():
    """The statements in float64 against autograd through torch's functions, and their 8-bit rounding against torch's."""
    g = torch.Generator().manual_seed(0)
    x, w, b, gr = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((7, 5), (4, 5), (4,), (7, 4)))
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = 1.3 * torch.nn.functional.gelu(0.4 * leaves[0] @ leaves[1].t() + leaves[2])
    want = (y.detach(), *torch.autograd.grad(y, leaves, gr))
    got = O.dense(x, w, b, None, "gelu", 1.3, 0.4, gr)
    assert all(torch.allclose(got[k][0], t, rtol=1e-12, atol=1e-13) for k, t in zip(("y", "dx", "dw", "db"), want))
    assert O.group_rows(torch.tensor([-3, 5, 2, 99]), 8) == [(0, 5), (5, 5), (5, 8)]
    v = torch.randn(50, 300, generator=g) * torch.exp(3 * torch.randn(50, 300, generator=g))
    q, scale = O.e4m3_rows(v.double())
    assert torch.equal(q, (v.double() / scale[:, None]).float().to(F8).double())


def test_rows_by_element():
    """Sorted and put back, on the CPU; gradients go the way back; ids outside are in no group."""
    from flashcart_amd.nn import ElementRows
    ids = torch.tensor([[2, 0, 1], [-1, 0, 5], [2, 2, 0]])
    rows = ElementRows(ids, 3)
    x = torch.randn(3, 3, 4, requires_grad=True)
    s = rows.sort(x)
    assert rows.offsets.tolist() == [1, 4, 5, 8]
    assert torch.equal(ids.reshape(-1)[rows.order], torch.tensor([-1, 0, 0, 0, 1, 2, 2, 2, 5]))
    assert torch.equal(rows.unsort(s).view_as(x), x)
    g = torch.randn(9, 4)
    (gx,) = torch.autograd.grad(s, x, g)
    assert torch.equal(gx.view(9, 4)[rows.order], g)
    assert torch.autograd.gradgradcheck(lambda t: rows.sort(t) ** 3, torch.randn(3, 3, 2, dtype=torch.float64, requires_grad=True))


def test_layers_refuse_other_activations():
    from flashcart_amd.nn import DenseLayer, ElementDenseLayer
    for make in (lambda: DenseLayer(4, 4, "relu"), lambda: ElementDenseLayer(2, 4, 4, "relu")):
        with pytest.raises(ValueError, match="activation must be None or one of"):
            make()
