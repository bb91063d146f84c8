"""The registered operators of ``flashcart_amd.nn.functional`` (``torch.ops.flashcart.embedding``, ``dropout_add``,
``gated_feed_forward`` and their backward passes). They are C++ operators over the C entry points
(``csrc/torch/node_ops.cpp``, ``libflashcart_torch.so``); here they are loaded and given their shape-only
implementations."""

from __future__ import annotations

import ctypes
import os

import torch

from flashcart_amd import _lib

ACTIVATIONS = {"silu": 0, "sigmoid": 1, "gelu": 2}

TORCH_LIB_PATH = os.path.join(os.path.dirname(_lib.LIB_PATH), "libflashcart_torch.so")


_loaded = False


def _load() -> None:
    global _loaded
    _lib.load()
    if not os.path.exists(TORCH_LIB_PATH):
        raise _lib.HipLibraryError(f"{TORCH_LIB_PATH} is missing: build it with `python -m flashcart_amd.build`.")
    torch.ops.load_library(TORCH_LIB_PATH)
    if ctypes.CDLL(TORCH_LIB_PATH).fct_bind(_lib.LIB_PATH.encode()) != 0:
        raise _lib.HipLibraryError(f"{_lib.LIB_PATH} lacks the node-wise entry points: build it again.")
    for name, fake in _FAKES.items():
        torch.library.register_fake(f"flashcart::{name}", fake)
    _loaded = True


def ops():
    """``torch.ops.flashcart`` with these operators."""
    if not _loaded:
        _load()
    return torch.ops.flashcart


def _contiguous(t, need=True):
    return torch.empty_like(t, memory_format=torch.contiguous_format) if need else t.new_empty(0)


def _embedding(ids, table, scale, padding):
    return table.new_empty((*ids.shape, table.shape[1]))


def _embedding_bwd(grad, ids, rows, scale, padding):
    return grad.new_empty(rows, grad.shape[-1])


def _dropout_add(x, residual, p, rng):
    return _contiguous(x)


def _dropout_draw(state):
    return torch.empty_like(state)


def _gated_feed_forward(x, w_in, w_out, act, act_scale, scale_in, scale_out, save):
    width, hidden = w_out.shape
    size = 0
    if save:  # hidden values (three bf16 parts each for float32) and two factors
        size = x.numel() // width * ((hidden + 7) // 8 * 8) * (14 if x.dtype == torch.float32 else 8)
    return _contiguous(x), x.new_empty(size, dtype=torch.uint8)


def _gated_feed_forward_bwd(grad, x, w_in, w_out, saved, act, act_scale, scale_in, scale_out, need_x, need_w_in,
                            need_w_out):
    return _contiguous(x, need_x), _contiguous(w_in, need_w_in), _contiguous(w_out, need_w_out)


_FAKES = {"embedding": _embedding, "embedding_bwd": _embedding_bwd, "dropout_add": _dropout_add,
          "dropout_draw": _dropout_draw, "gated_feed_forward": _gated_feed_forward, "gated_feed_forward_bwd": _gated_feed_forward_bwd}

# With the import, so that a compiled function never meets the loading. Where it fails (not built, built for another torch)
# the first call says why; the rest of the package does not need it.
if os.path.exists(TORCH_LIB_PATH) and os.path.exists(_lib.LIB_PATH):
    try:
        _load()
    except (OSError, AttributeError, _lib.HipLibraryError):
        pass
