"""Node-wise operators without a GPU: the generator's published answers, refusals, shapes of fake tensors."""

import numpy as np
import pytest
import torch

from flashcart_amd.nn import functional as F
from oracle import node_ops as O


@pytest.mark.parametrize("word,key,want", [
    (0, 0, "6627e8d5 e169c58d bc57ac4c 9b00dbd8"),
    (0xFFFFFFFF, 0xFFFFFFFF, "408f276d 41c83b0e a20bc7c6 6d5451fd"),
])
def test_philox_known_answers(word, key, want):
    got = O.philox4x32(np.full((1, 4), word, dtype=np.uint64), (key, key))[0]
    assert " ".join(f"{int(v):08x}" for v in got) == want


def test_cpu_tensors_are_refused():
    table, rng = torch.zeros(3, 4), torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        F.embedding(torch.zeros(2, dtype=torch.int64), table)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        F.gated_feed_forward(torch.zeros(2, 4), torch.zeros(6, 4), torch.zeros(4, 3))
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        F.dropout_add(table, None, 0.5, rng)


@pytest.mark.parametrize("call,error", [
    (lambda: F.embedding(torch.zeros(2), torch.zeros(3, 4)), "int64 or int32"),
    (lambda: F.embedding(torch.zeros(2, dtype=torch.int64), torch.zeros(3, 4), padding_idx=3), "outside the table"),
    (lambda: F.embedding(torch.zeros(2, dtype=torch.int64), torch.zeros(3, 4), padding_idx=-4), "outside the table"),
    (lambda: F.embedding(torch.zeros(2, dtype=torch.int64), torch.zeros(3, 4, dtype=torch.float64)), "float32, bfloat16"),
    (lambda: F.dropout_add(torch.zeros(3, dtype=torch.int32), None, 0.5, torch.zeros(2)), "float32, bfloat16"),
])
def test_arguments_are_refused(call, error):
    with pytest.raises((TypeError, ValueError), match=error):
        call()


def test_fake_tensors_have_the_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        ids, table = torch.empty(2, 5, dtype=torch.int64), torch.empty(7, 3, dtype=torch.bfloat16)
        assert F.embedding(ids, table).shape == (2, 5, 3)
        x = torch.empty(4, 6, dtype=torch.float16)
        w_in, w_out = torch.empty(20, 6, dtype=torch.float16, requires_grad=True), torch.empty(6, 10, dtype=torch.float16)
        assert F.gated_feed_forward(x, w_in, w_out).shape == (4, 6)
        assert F.dropout_add(x, x, 0.1, torch.empty(2, dtype=torch.int64)).shape == (4, 6)


def test_library_refuses_bad_arguments():
    """Status codes of the C entry points, decided before anything is launched."""
    from flashcart_amd import _lib
    lib = _lib.load()
    bad_desc, shape, null, workspace = 1, 4, 5, 6
    assert lib.fc_embedding_fwd(3, 1, 1, 1, 1, 1, 1.0, 1, None) == bad_desc
    assert lib.fc_embedding_fwd(0, -1, 1, 1, None, None, 1.0, None, None) == shape
    assert lib.fc_embedding_fwd(0, 1, 0, 1, None, None, 1.0, None, None) == shape
    assert lib.fc_embedding_fwd(0, 1, 1, 1, None, None, 1.0, None, None) == null
    assert lib.fc_embedding_bwd_workspace(0, 1 << 31, 4, 4) == -shape
    need = lib.fc_embedding_bwd_workspace(1, 100, 7, 16)
    assert need > 0
    assert lib.fc_embedding_bwd(1, 100, 7, 16, 16, 16, 1.0, -1, 16, 16, need - 1, None) == workspace
    for p in (-0.1, 1.1, float("nan")):
        assert lib.fc_dropout_add(0, 1, 16, None, p, 16, 16, None) == bad_desc
    assert lib.fc_dropout_add(0, 1, 16, None, 0.5, None, 16, None) == null
    desc = _lib.FfnDesc(0, 0, 8, 16, 1, 1.0, 1.0, 1.0)
    assert lib.fc_ffn_saved(desc, 3) == 3 * 16 * 14 and lib.fc_ffn_saved(desc, -1) == -shape
    assert lib.fc_ffn_fwd(desc, 3, 18, 16, 16, 16, 16, 16, 1 << 20, None) == bad_desc  # not aligned
    desc.aligned = 0  # every operand is copied
    size = lib.fc_ffn_fwd_workspace(desc, 3, 1)
    assert size > 0 and lib.fc_ffn_fwd_workspace(desc, 3, 0) > size
    assert lib.fc_ffn_fwd(desc, 3, 16, 16, 16, 16, 16, 16, size - 1, None) == workspace
    assert lib.fc_ffn_fwd(desc, 3, 16, 16, 16, None, 16, 16, size, None) == null
    assert lib.fc_ffn_bwd(desc, 3, 16, 16, 16, 16, None, 16, None, None, 16, 1 << 20, None) == null
    for bad, code in ((dict(dtype=3), bad_desc), (dict(act=3), bad_desc), (dict(width=0), shape),
                      (dict(hidden=(1 << 20) + 1), shape)):
        fields = dict(dtype=1, act=0, width=8, hidden=16, aligned=1, act_scale=1.0, scale_in=1.0, scale_out=1.0)
        assert lib.fc_ffn_saved(_lib.FfnDesc(**{**fields, **bad}), 3) == -code
    assert lib.fc_dropout_add(0, 0, None, None, 0.5, None, None, None) == 0


def test_compilers_see_the_operators():
    """One graph with the operators themselves in it (which then end in their own error on the CPU)."""
    seen = []

    def backend(graph, inputs):
        seen.extend(str(n.target) for n in graph.graph.nodes if n.op == "call_function")
        return graph.forward

    def block(ids, table, w_in, w_out, rng):
        e = F.embedding(ids, table, 2.0, 0)
        return F.dropout_add(F.gated_feed_forward(e, w_in, w_out), e, 0.1, rng)

    rng = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        torch.compile(block, backend=backend, fullgraph=True)(rng, torch.zeros(3, 4), torch.zeros(6, 4),
                                                              torch.zeros(4, 3), rng)
    for name in ("embedding", "gated_feed_forward", "dropout_add"):
        assert any(f"flashcart.{name}.default" in t for t in seen)
