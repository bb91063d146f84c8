"""Registered operators of the node-wise functions (``flashcart_amd.nn.functional``): embedding and residual dropout.
float32, bfloat16 and float16 tensors on a ROCm device; every value is formed in float32 and rounded once.
"""

from __future__ import annotations

from typing import Optional

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
