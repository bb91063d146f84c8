"""Node-wise functions in float32, bfloat16 and float16: embedding lookup, residual dropout.

They have no counterpart among the reference's kernels (it composes torch operations). Each is a registered operator
(``torch.ops.flashcart.*``) with an autograd formula, runs on the current stream and allocates through torch, so it can
be captured into a graph. There is no CPU path. Values are formed in float32 and rounded once to the tensors' type.
"""

from typing import Optional

import torch

from flashcart_amd.nn import _node_ops
from flashcart_amd.o3._ops import param_alias

__all__ = ["dropout_add", "embedding"]


def embedding(ids: torch.Tensor, table: torch.Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * table[ids]``.

    Args:
        ids: int64 or int32, any shape. An index outside the table gives a row of NaN (a kernel cannot raise) and takes
            no part in the gradient.
        table: (rows, width).
        scale: factor of every row.
        padding_idx: row that gets no gradient; negative counts from the end.

    Returns:
        (*ids.shape, width) in the table's type. The table's gradient adds the rows of each index in the order of the
        tokens, in float32: it is the same in every run.
    """
    if ids.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"`ids` must be int64 or int32, got {ids.dtype}.")
    rows = table.shape[0] if table.dim() == 2 else 0
    padding = -1
    if padding_idx is not None:
        padding = padding_idx + rows if padding_idx < 0 else padding_idx
        if not 0 <= padding < rows:
            raise ValueError(f"padding_idx={padding_idx} is outside the table of {rows} rows.")
    return _node_ops.embedding(ids, param_alias(table), float(scale), padding)


def dropout_add(x: torch.Tensor, residual: Optional[torch.Tensor], p: float, rng: torch.Tensor) -> torch.Tensor:
    """``residual + dropout(x, p)`` from a counter-based generator, without a stored mask.

    Element e is kept when word e % 4 of the Philox4x32-10 block of counter (e // 4, offset) and key ``seed`` is at least
    floor(p 2^32); the backward pass forms the mask again.

    Args:
        x: any shape.
        residual: same shape and type, or None.
        p: probability of dropping an element, in [0, 1].
        rng: int64 tensor (seed, offset) on x's device. The caller advances the offset from call to call (on the device
            where the call is captured into a graph): the same pair gives the same mask.
    """
    return _node_ops.dropout_add(x, residual, float(p), rng)
