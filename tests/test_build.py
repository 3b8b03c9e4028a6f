"""CPU tests of the build: what is rebuilt when, and that the library does not depend on the module of the tensor calls."""
import os
import subprocess

import pytest

from bullet_b200 import build as b


@pytest.fixture
def tools(monkeypatch, tmp_path):
    """The build's outputs in a folder of their own, and compilers that note their calls: they write what they are asked for unless told to
    fail."""
    calls, broken = [], set()

    def run(cmd, **kw):
        tool = "library" if cmd[cmd.index("-o") + 1] == b.LIB else "module"
        calls.append(tool)
        if tool in broken:
            return subprocess.CompletedProcess(cmd, 1, "", "an error\n")
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(b, "LIB", str(tmp_path / "library.so"))
    monkeypatch.setattr(b, "TENSOR_CALLS", str(tmp_path / "module.so"))
    if hasattr(b, "MADE_FOR"):
        monkeypatch.setattr(b, "MADE_FOR", str(tmp_path / "module.made_for"))
    monkeypatch.setattr(b.subprocess, "run", run)
    return calls, broken


def test_what_is_up_to_date_is_not_built_again(tools):
    calls, _ = tools
    assert b.build() == b.LIB and calls == ["library", "module"]
    assert b.build() == b.LIB and calls == ["library", "module"]
    assert b.build(force=True) == b.LIB and calls == 2 * ["library", "module"]


def test_a_module_that_cannot_be_built_leaves_the_library(tools, capsys):
    calls, broken = tools
    broken.add("module")
    assert b.build() == b.LIB and os.path.exists(b.LIB) and not os.path.exists(b.TENSOR_CALLS)
    assert "ops is not built" in capsys.readouterr().err
    assert b.build() == b.LIB and calls == ["library", "module", "module"]  # (the library once)
    broken.clear()
    assert b.build() == b.LIB and os.path.exists(b.TENSOR_CALLS) and calls == ["library"] + 3 * ["module"]


def test_a_library_that_cannot_be_built_is_an_error(tools):
    calls, broken = tools
    broken.add("library")
    with pytest.raises(RuntimeError, match="nvcc failed"):
        b.build()
    assert calls == ["library"]


@pytest.mark.parametrize("missing", ["libtorch_cuda.so", "libc10_cuda.so", "Python.h"])
def test_what_the_module_needs_and_is_not_there(tools, monkeypatch, capsys, missing):
    calls, _ = tools
    there = os.path.exists
    monkeypatch.setattr(b.os.path, "exists", lambda p: there(p) and os.path.basename(str(p)) != missing)
    assert b.build() == b.LIB and calls == ["library"]
    assert missing in capsys.readouterr().err


def test_without_torch_nothing_but_the_library_is_wanted(tools, monkeypatch):
    calls, _ = tools
    monkeypatch.setattr(b, "_torch_dir", lambda: None)
    for _ in range(2):
        assert b.build() == b.LIB
    assert calls == ["library"]


def test_another_torch_has_the_module_built_again_and_no_module_of_the_old_one_stays(tools, monkeypatch):
    calls, broken = tools
    b.build()
    version = b.importlib.metadata.version
    monkeypatch.setattr(b.importlib.metadata, "version", lambda name: "99.0" if name == "torch" else version(name))
    broken.add("module")
    assert b.build() == b.LIB and calls == ["library", "module", "module"] and not os.path.exists(b.TENSOR_CALLS)
    broken.clear()
    b.build()
    b.build()
    assert calls == ["library"] + 3 * ["module"]


def test_each_output_is_as_old_as_its_own_sources(tools):
    calls, _ = tools
    b.build()
    os.utime(b.TENSOR_CALLS, (1, 1))  # (older than its source)
    b.build()
    assert calls == ["library", "module", "module"]
    os.utime(b.LIB, (1, 1))
    b.build()
    assert calls == ["library", "module", "module", "library"]
