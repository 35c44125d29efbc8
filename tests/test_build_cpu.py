"""build.py's decisions about _serving.so, which is compiled against one PyTorch
and one interpreter: rebuilt when either is another, left out without PyTorch.
Nothing is compiled here."""
import importlib.util
import os

import pytest
import torch

import vit_cuda
from vit_cuda import serving

PKG = os.path.dirname(os.path.dirname(os.path.abspath(vit_cuda.__file__)))


@pytest.fixture
def builder(monkeypatch, tmp_path):
    """The build module with its outputs elsewhere and a compiler that writes what it
    was asked for; `builder.calls` counts its runs."""
    spec = importlib.util.spec_from_file_location("build_under_test", os.path.join(PKG, "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    b.calls = []

    class Done:
        returncode, stdout, stderr = 0, "", ""

    def run(cmd, **kw):
        b.calls.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write(" ".join(cmd))
        return Done

    monkeypatch.setattr(b.subprocess, "run", run)
    monkeypatch.setattr(b, "nvcc", lambda: "/usr/local/cuda/bin/nvcc")
    monkeypatch.setattr(b, "OBJ_DIR", str(tmp_path / "obj"))
    monkeypatch.setattr(b, "BINDINGS_LIB", str(tmp_path / "_serving.so"))
    monkeypatch.setattr(b, "BINDINGS_STAMP", str(tmp_path / "obj" / "built_for"), raising=False)
    return b


def test_rebuilt_for_another_pytorch_or_python(builder, monkeypatch, tmp_path):
    builder.build_bindings()
    builder.build_bindings()
    assert len(builder.calls) == 1  # up to date
    # another PyTorch in the same place: no file of this repository is newer
    other = tmp_path / "torch"
    other.mkdir()
    (other / "version.py").write_text("__version__ = '9.9.9'\n")

    class Spec:
        submodule_search_locations = [str(other)]

    with monkeypatch.context() as m:
        m.setattr(builder.importlib.util, "find_spec", lambda name: Spec)
        builder.build_bindings()
        builder.build_bindings()
    assert len(builder.calls) == 2
    builder.build_bindings()
    assert len(builder.calls) == 3
    with monkeypatch.context() as m:
        get = builder.sysconfig.get_config_var
        m.setattr(builder.sysconfig, "get_config_var",
                  lambda n: ".cpython-399.so" if n == "EXT_SUFFIX" else get(n))
        builder.build_bindings()
    assert len(builder.calls) == 4


def test_c_library_without_pytorch(builder, monkeypatch, capsys):
    monkeypatch.setattr(builder.importlib.util, "find_spec", lambda name: None)
    monkeypatch.setattr(builder, "build_library", lambda *a: "lib")
    assert builder.build() == "lib"
    assert builder.calls == [] and "PyTorch" in capsys.readouterr().err


def test_module_of_another_pytorch_is_refused(monkeypatch):
    module = serving.direct()
    assert module.BUILT_FOR == torch.__version__
    monkeypatch.setattr(serving, "_ops", None)
    monkeypatch.setattr(module, "BUILT_FOR", "9.9.9")
    with pytest.raises(ImportError, match="build.py"):
        serving.direct()
