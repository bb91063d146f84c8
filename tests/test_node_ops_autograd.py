"""What the autograd formulas of the node-wise operators do around their kernels, seen on tensors without memory."""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

from flashcart_amd.nn import functional as F

OPERATORS = ["embedding", "embedding_bwd", "dropout_add", "residual", "gated_feed_forward", "w_out"]


def _call(name):
    """The operator as a function of one differentiable argument, and that argument."""
    ids, rng = torch.zeros(3, dtype=torch.int64), torch.zeros(2, dtype=torch.int64)
    x, w_in, w_out = torch.empty(5, 4), torch.empty(12, 4), torch.empty(4, 6)
    return {
        "embedding": (lambda t: F.embedding(ids, t, 2.0, 0), torch.empty(7, 4)),
        "embedding_bwd": (lambda t: torch.ops.flashcart.embedding_bwd(t, ids, 7, 2.0, -1), torch.empty(3, 4)),
        "dropout_add": (lambda t: F.dropout_add(t, None, 0.5, rng), x),
        "residual": (lambda t: F.dropout_add(x, t, 0.5, rng), torch.empty(5, 4)),
        "gated_feed_forward": (lambda t: F.gated_feed_forward(t, w_in, w_out), x),
        "w_out": (lambda t: F.gated_feed_forward(x, w_in, t), w_out),
    }[name]


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("enabled", [False, True])
@pytest.mark.parametrize("name", OPERATORS)
def test_forward_mode_is_refused(name, enabled, recorded):
    """A tangent is never dropped: forward-mode derivatives, which the operators lack, raise."""
    with FakeTensorMode(), forward_ad.dual_level(), torch.set_grad_enabled(enabled):
        call, t = _call(name)
        dual = forward_ad.make_dual(t.requires_grad_(recorded), torch.empty_like(t))
        with pytest.raises(RuntimeError, match="jvp is not implemented"):
            call(dual)
        assert call(t).requires_grad == (enabled and recorded)  # (the level alone refuses nothing)


@pytest.mark.parametrize("name", OPERATORS)
def test_functional_forward_mode_is_refused(name):
    with FakeTensorMode():
        call, t = _call(name)
        with pytest.raises(RuntimeError, match="functorch transforms"):
            torch.func.jvp(call, (t,), (torch.empty_like(t),))


class _Calls(TorchDispatchMode):
    """The operators that run, without queries of properties."""

    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace != "prim":
            self.names.append(func.name())
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("name", OPERATORS)
def test_backward_passes_run_their_operator_alone(name):
    """No zeros for outputs without a gradient (the block's kept values are the largest tensor of a training step)."""
    with FakeTensorMode():
        call, t = _call(name)
        out = call(t.requires_grad_())
        grad = torch.empty_like(out)
        with _Calls() as calls:
            torch.autograd.grad(out, t, grad)
    if name == "residual":
        assert calls.names == []
    elif name == "embedding_bwd":  # its cotangent is looked up, but for ids that add to no row
        assert "flashcart::embedding" in calls.names and not any("zeros" in n for n in calls.names)
    else:
        assert calls.names == [{"embedding": "flashcart::embedding_bwd", "dropout_add": "flashcart::dropout_add"}.get(
            name, "flashcart::gated_feed_forward_bwd")]


def test_block_without_a_gradient_of_its_output():
    """A pass that reaches the block with no gradient of y gives none to its arguments."""
    with FakeTensorMode():
        call, t = _call("gated_feed_forward")

        class Stop(torch.autograd.Function):
            @staticmethod
            def forward(ctx, x):
                return x.clone()

            @staticmethod
            def backward(ctx, grad):
                return None

        out = Stop.apply(call(t.requires_grad_()))
        ones = torch.empty_like(out)
        with _Calls() as calls:
            (grad,) = torch.autograd.grad(out, t, ones, allow_unused=True)
        assert grad is None and calls.names == []


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,width,hidden", [(1, 1, 1), (7, 24, 40), (600, 520, 523), (2000, 1024, 1024), (0, 8, 8)])
def test_kept_bytes_of_fake_tensors(n, width, hidden, dtype):
    """The shape-only operator keeps as many bytes as the library asks for, in every form of the products."""
    from flashcart_amd import _lib
    code = [torch.float32, torch.bfloat16, torch.float16].index(dtype)
    want = _lib.load().fc_ffn_saved(_lib.FfnDesc(code, 0, width, hidden, 1, 1.0, 1.0, 1.0), n)
    with FakeTensorMode():
        x, w_in, w_out = (torch.empty(*s, dtype=dtype) for s in ((n, width), (2 * hidden, width), (width, hidden)))
        saved = torch.ops.flashcart.gated_feed_forward(x, w_in, w_out, 0, 1.0, 1.0, 1.0, True)[1]
    assert saved.numel() == want
