"""What the incremental build takes for current."""

import os

import pytest
import torch

from flashcart_amd import build
from flashcart_amd.codegen import emit_hip


@pytest.fixture
def steps(tmp_path, monkeypatch):
    """A build of empty files in a folder of its own; the list of what it ran."""
    ran = []

    def touch(path):
        open(path, "w").close()

    def compiled(src, gen, build_dir):
        ran.append("compile")
        return src

    monkeypatch.setattr(build, "BUILD", str(tmp_path / "objects"))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "kernels.so"))
    monkeypatch.setattr(build, "TORCH_LIB", str(tmp_path / "operators.so"))
    monkeypatch.setattr(build, "_sources", lambda: [os.path.join(build.CSRC, "fc_dropout.hip")])
    monkeypatch.setattr(build, "_compile", compiled)
    monkeypatch.setattr(build, "_link", lambda objs, lib: (ran.append("link"), touch(lib)))
    monkeypatch.setattr(build, "_build_torch", lambda: (ran.append("operators"), touch(build.TORCH_LIB)))
    monkeypatch.setattr(emit_hip, "write_all", lambda gen, l_max: None)
    return ran


def _run(steps, **kwargs):
    del steps[:]
    build.build(l_max=3, **kwargs)
    return sorted(steps)


def test_incremental_build(steps, monkeypatch):
    everything = ["compile", "link", "operators"]
    assert _run(steps, force=False) == everything
    assert _run(steps, force=False) == []
    assert _run(steps, force=True) == everything
    # the operators' library holds code for one torch
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert _run(steps, force=False) == ["operators"]
    assert _run(steps, force=False) == []
    os.remove(build.TORCH_LIB)
    assert _run(steps, force=False) == ["operators"]
    os.remove(build.LIB)
    assert _run(steps, force=False) == ["compile", "link"]
    monkeypatch.setattr(build, "CFLAGS", [*build.CFLAGS, "-DOTHER"])
    assert _run(steps, force=False) == ["compile", "link"]


def test_failed_operators_are_not_taken_for_built(steps, monkeypatch):
    def fails():
        raise RuntimeError("g++ failed")

    with monkeypatch.context() as m:
        m.setattr(build, "_build_torch", fails)
        with pytest.raises(RuntimeError, match="g\\+\\+ failed"):
            build.build(l_max=3, force=False)
    assert _run(steps, force=False) == ["compile", "link", "operators"]
