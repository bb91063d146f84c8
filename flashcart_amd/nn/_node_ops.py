"""Registered operators of the node-wise functions (``flashcart_amd.nn.functional``): embedding, gated feed-forward
block, residual dropout. float32, bfloat16 and float16 tensors on a ROCm device; values are formed in float32.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from flashcart_amd import _lib
from flashcart_amd.o3._ops import _lib_call, _register_autograd, operator

Tensor = torch.Tensor


def _code(name: str, t: Tensor) -> int:
    if t.dtype not in _lib.NODE_DTYPES:
        raise TypeError(f"`{name}` must be float32, bfloat16 or float16, got {t.dtype}.")
    return _lib.NODE_DTYPES[t.dtype]


def _same_device(first: Tensor, **others: Optional[Tensor]) -> None:
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise RuntimeError(f"`{name}` is on {t.device}, the other arguments are on {first.device}.")


def _workspace(like: Tensor, size: int) -> Tensor:
    """``size`` bytes, or the error that a workspace query answers with a negative size."""
    if size < 0:
        _lib.check(-size, "workspace query")
    return like.new_empty(size, dtype=torch.uint8)


# ---------------------------------------------------------------------------
# Embedding
# ---------------------------------------------------------------------------

@operator("flashcart::embedding")
def embedding(ids: Tensor, table: Tensor, scale: float, padding: int) -> Tensor:
    """``scale * table[ids]``; ids of any shape, ``padding``: the row without a gradient (-1: none)."""
    code = _code("table", table)
    table = _lib.contig("table", table, table.dtype)
    if table.dim() != 2 or table.shape[0] < 1 or table.shape[1] < 1:
        raise ValueError(f"embedding: the table must be (rows, width) and not empty, got {tuple(table.shape)}.")
    if ids.dtype == torch.int32:
        ids = ids.long()
    ids = _lib.contig("ids", ids, torch.int64)
    _same_device(table, ids=ids)
    out = table.new_empty((*ids.shape, table.shape[1]))
    _lib_call("fc_embedding_fwd", code, ids.numel(), table.shape[0], table.shape[1], ids.data_ptr(), table.data_ptr(),
              float(scale), out.data_ptr(), _lib.stream_of(table))
    return out


@embedding.register_fake
def _(ids, table, scale, padding):
    return table.new_empty((*ids.shape, table.shape[1]))


@operator("flashcart::embedding_bwd")
def embedding_bwd(grad: Tensor, ids: Tensor, rows: int, scale: float, padding: int) -> Tensor:
    """The table's gradient: ``scale`` times the sum of each index's gradient rows, in a fixed order."""
    code = _code("grad", grad)
    g = _lib.contig("grad", grad, grad.dtype)
    if ids.dtype == torch.int32:
        ids = ids.long()
    ids = _lib.contig("ids", ids, torch.int64)
    if g.dim() < 1 or g.shape[:-1] != ids.shape:
        raise ValueError(f"embedding_bwd: grad {tuple(g.shape)} does not match ids {tuple(ids.shape)}.")
    _same_device(g, ids=ids)
    n, width = ids.numel(), g.shape[-1]
    out = g.new_empty(rows, width)
    size = _lib.load().fc_embedding_bwd_workspace(code, n, rows, width)
    ws = _workspace(g, size)
    _lib_call("fc_embedding_bwd", code, n, rows, width, ids.data_ptr(), g.data_ptr(), float(scale), int(padding),
              out.data_ptr(), ws.data_ptr(), size, _lib.stream_of(g))
    return out


@embedding_bwd.register_fake
def _(grad, ids, rows, scale, padding):
    return grad.new_empty(rows, grad.shape[-1])


def _embedding_setup(ctx, inputs, output):
    ids, table, scale, padding = inputs
    ctx.save_for_backward(ids)
    ctx.cfg = (table.shape[0], float(scale), int(padding))


def _embedding_backward(ctx, grad):
    (ids,) = ctx.saved_tensors
    return None, embedding_bwd(grad, ids, *ctx.cfg) if ctx.needs_input_grad[1] else None, None, None


def _embedding_bwd_setup(ctx, inputs, output):
    grad, ids, rows, scale, padding = inputs
    ctx.save_for_backward(ids)
    ctx.cfg = (rows, float(scale), int(padding))


def _embedding_dbwd(ctx, cot):
    """The table's gradient is linear in ``grad``: the rows that an id adds to, looked up in the cotangent (zero for
    the padding row and for ids outside the table, which add to none)."""
    (ids,) = ctx.saved_tensors
    if not ctx.needs_input_grad[0]:
        return None, None, None, None, None
    rows, scale, padding = ctx.cfg
    out = embedding(ids.clamp(0, rows - 1), cot, scale, padding)
    dead = (ids < 0) | (ids >= rows) | (ids == padding)
    return out.masked_fill(dead.unsqueeze(-1), 0.0), None, None, None, None


_register_autograd(embedding, _embedding_backward, _embedding_setup)
_register_autograd(embedding_bwd, _embedding_dbwd, _embedding_bwd_setup)


# ---------------------------------------------------------------------------
# Residual dropout
# ---------------------------------------------------------------------------

@operator("flashcart::dropout_add")
def dropout_add(x: Tensor, residual: Optional[Tensor], p: float, rng: Tensor) -> Tensor:
    """``residual + keep * x / (1 - p)``; ``rng``: (seed, offset), two int64 on the device."""
    code = _code("x", x)
    x = _lib.contig("x", x, x.dtype)
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"dropout_add: residual {tuple(residual.shape)} and x {tuple(x.shape)} differ in shape.")
        residual = _lib.contig("residual", residual, x.dtype)
    if rng.numel() != 2:
        raise ValueError(f"dropout_add: rng must hold a seed and an offset, got {tuple(rng.shape)}.")
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout_add: p must be in [0, 1], got {p}.")
    rng = _lib.contig("rng", rng, torch.int64)
    _same_device(x, residual=residual, rng=rng)
    out = torch.empty_like(x)
    _lib_call("fc_dropout_add", code, x.numel(), x.data_ptr(), _lib.ptr(residual), float(p), rng.data_ptr(),
              out.data_ptr(), _lib.stream_of(x))
    return out


@dropout_add.register_fake
def _(x, residual, p, rng):
    return torch.empty_like(x, memory_format=torch.contiguous_format)


def _dropout_setup(ctx, inputs, output):
    x, residual, p, rng = inputs
    ctx.save_for_backward(rng)
    ctx.p = float(p)


def _dropout_backward(ctx, grad):
    (rng,) = ctx.saved_tensors
    gx = dropout_add(grad, None, ctx.p, rng) if ctx.needs_input_grad[0] else None
    return gx, grad if ctx.needs_input_grad[1] else None, None, None


_register_autograd(dropout_add, _dropout_backward, _dropout_setup)


# ---------------------------------------------------------------------------
# Gated feed-forward block
# ---------------------------------------------------------------------------

ACTIVATIONS = {"silu": 0, "sigmoid": 1, "gelu": 2}


def _ffn_desc(what: str, rows: Tensor, w_in: Tensor, w_out: Tensor, act: int, act_scale: float, scale_in: float,
              scale_out: float):
    """(descriptor without ``aligned``, rows of the block)."""
    code = _code("x", rows)
    if w_out.dim() != 2 or w_in.dim() != 2 or w_in.shape[0] != 2 * w_out.shape[1] or w_in.shape[1] != w_out.shape[0]:
        raise ValueError(f"{what}: w_in {tuple(w_in.shape)} and w_out {tuple(w_out.shape)} are not (2 hidden, width) "
                         "and (width, hidden).")
    width, hidden = w_out.shape
    if width < 1 or hidden < 1 or rows.dim() < 1 or rows.shape[-1] != width:
        raise ValueError(f"{what}: rows {tuple(rows.shape)} do not match weights of width {width}, hidden {hidden}.")
    if act not in (0, 1, 2):
        raise ValueError(f"{what}: act must be 0 (silu), 1 (sigmoid) or 2 (gelu), got {act}.")
    desc = _lib.FfnDesc(code, act, width, hidden, 0, float(act_scale), float(scale_in), float(scale_out))
    return desc, rows.numel() // width


def _aligned(*tensors: Tensor) -> int:
    return int(all(t.data_ptr() % 16 == 0 for t in tensors))


@operator("flashcart::gated_feed_forward")
def gated_feed_forward(x: Tensor, w_in: Tensor, w_out: Tensor, act: int, act_scale: float, scale_in: float,
                       scale_out: float, save: bool) -> Tuple[Tensor, Tensor]:
    """(y, what the backward pass needs besides the inputs, empty unless ``save``)."""
    desc, n = _ffn_desc("gated_feed_forward", x, w_in, w_out, act, act_scale, scale_in, scale_out)
    x = _lib.contig("x", x, x.dtype)
    w_in, w_out = _lib.contig("w_in", w_in, x.dtype), _lib.contig("w_out", w_out, x.dtype)
    _same_device(x, w_in=w_in, w_out=w_out)
    desc.aligned = _aligned(x, w_in, w_out)
    lib = _lib.load()
    y = torch.empty_like(x)
    saved = _workspace(x, lib.fc_ffn_saved(desc, n) if save else 0)
    size = lib.fc_ffn_fwd_workspace(desc, n, int(save))
    ws = _workspace(x, size)
    _lib_call("fc_ffn_fwd", desc, n, x.data_ptr(), w_in.data_ptr(), w_out.data_ptr(), y.data_ptr(),
              saved.data_ptr() if save and n else None, ws.data_ptr(), size, _lib.stream_of(x))
    return y, saved


@gated_feed_forward.register_fake
def _(x, w_in, w_out, act, act_scale, scale_in, scale_out, save):
    desc, n = _ffn_desc("gated_feed_forward", x, w_in, w_out, act, act_scale, scale_in, scale_out)
    planes, factors = (3, 8) if x.dtype == torch.float32 else (1, 6)
    size = n * -(-w_out.shape[1] // 8) * 8 * (2 * planes + factors) if save else 0
    return torch.empty_like(x, memory_format=torch.contiguous_format), x.new_empty(size, dtype=torch.uint8)


@operator("flashcart::gated_feed_forward_bwd")
def gated_feed_forward_bwd(grad: Tensor, x: Tensor, w_in: Tensor, w_out: Tensor, saved: Tensor, act: int,
                           act_scale: float, scale_in: float, scale_out: float, need_x: bool, need_w_in: bool,
                           need_w_out: bool) -> Tuple[Tensor, Tensor, Tensor]:
    """(gradient of x, of w_in, of w_out), empty where not needed."""
    desc, n = _ffn_desc("gated_feed_forward_bwd", x, w_in, w_out, act, act_scale, scale_in, scale_out)
    if grad.shape != x.shape:
        raise ValueError(f"gated_feed_forward_bwd: grad {tuple(grad.shape)} and x {tuple(x.shape)} differ in shape.")
    x = _lib.contig("x", x, x.dtype)
    g = _lib.contig("grad", grad, x.dtype)
    w_in, w_out = _lib.contig("w_in", w_in, x.dtype), _lib.contig("w_out", w_out, x.dtype)
    saved = _lib.contig("saved", saved, torch.uint8)
    _same_device(x, grad=g, w_in=w_in, w_out=w_out, saved=saved)
    lib = _lib.load()
    desc.aligned = _aligned(g, x, w_in, w_out)
    if saved.numel() != lib.fc_ffn_saved(desc, n):
        raise ValueError(f"gated_feed_forward_bwd: saved holds {saved.numel()} bytes, not the {lib.fc_ffn_saved(desc, n)} "
                         "of a forward pass with save=True.")
    if saved.data_ptr() % 16:
        saved = saved.clone()
    empty = torch.zeros_like if n == 0 else torch.empty_like
    gx, gwi, gwo = (empty(t) if need else t.new_empty(0)
                    for t, need in ((x, need_x), (w_in, need_w_in), (w_out, need_w_out)))
    if n == 0:
        return gx, gwi, gwo
    size = lib.fc_ffn_bwd_workspace(desc, n, int(need_x), int(need_w_in), int(need_w_out))
    ws = _workspace(x, size)
    _lib_call("fc_ffn_bwd", desc, n, g.data_ptr(), x.data_ptr(), w_in.data_ptr(), w_out.data_ptr(), saved.data_ptr(),
              gx.data_ptr() if need_x else None, gwi.data_ptr() if need_w_in else None,
              gwo.data_ptr() if need_w_out else None, ws.data_ptr(), size, _lib.stream_of(x))
    return gx, gwi, gwo


@gated_feed_forward_bwd.register_fake
def _(grad, x, w_in, w_out, saved, act, act_scale, scale_in, scale_out, need_x, need_w_in, need_w_out):
    return tuple(torch.empty_like(t, memory_format=torch.contiguous_format) if need else t.new_empty(0)
                 for t, need in ((x, need_x), (w_in, need_w_in), (w_out, need_w_out)))


def _ffn_setup(ctx, inputs, output):
    x, w_in, w_out = inputs[:3]
    ctx.save_for_backward(x, w_in, w_out, output[1])
    ctx.cfg = inputs[3:7]
    ctx.save = inputs[7]
    ctx.mark_non_differentiable(output[1])


def _ffn_backward(ctx, grad, _):
    x, w_in, w_out, saved = ctx.saved_tensors
    need = [bool(v) for v in ctx.needs_input_grad[:3]]
    if not any(need):
        return (None,) * 8
    if not ctx.save:
        raise RuntimeError("gated_feed_forward was called with save=False: its gradients cannot be formed.")
    grads = gated_feed_forward_bwd(grad, x, w_in, w_out, saved, *ctx.cfg, *need)
    return (*(g if n else None for g, n in zip(grads, need)), *(None,) * 5)


def _ffn_bwd_setup(ctx, inputs, output):
    pass


def _ffn_dbwd(ctx, *cots):
    raise NotImplementedError("second derivatives of gated_feed_forward are not provided "
                              "(its backward pass was run with create_graph=True).")


_register_autograd(gated_feed_forward, _ffn_backward, _ffn_setup)
_register_autograd(gated_feed_forward_bwd, _ffn_dbwd, _ffn_bwd_setup)
