"""The build: the library needs no torch, the binding belongs to the torch it was built against."""
import os
import sys

import pytest

from proteinpredictmachinelearning_b200 import _lib
from proteinpredictmachinelearning_b200 import build as b


@pytest.fixture
def no_binding(monkeypatch, tmp_path):
    """A tree with the library and without the binding."""
    monkeypatch.setattr(b, "TORCH_BINDING", str(tmp_path / "ppml_b200_torch.so"))
    monkeypatch.setattr(b, "TORCH_STAMP", str(tmp_path / "ppml_b200_torch.txt"))
    return tmp_path


def test_library_builds_without_torch(lib, no_binding, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    assert b.build() == b.LIB
    assert "torch is not installed" in capsys.readouterr().err and not os.listdir(no_binding)


def test_library_builds_beside_a_torch_without_cuda(lib, no_binding, monkeypatch, capsys):
    torch = pytest.importorskip("torch")
    monkeypatch.setattr(torch.version, "cuda", None)
    assert b.build() == b.LIB
    assert "no CUDA" in capsys.readouterr().err and not os.listdir(no_binding)


def test_binding_is_built_again_for_another_torch(no_binding, monkeypatch):
    pytest.importorskip("torch")
    made = []

    def run(cmd):
        made.append(cmd)
        open(b.TORCH_BINDING, "w").close()
    b.build_torch_binding(run)
    b.build_torch_binding(run)
    assert len(made) == 1
    monkeypatch.setattr(b, "_installed_torch", lambda: "torch 9.9.9, cpython-399")
    b.build_torch_binding(run)
    b.build_torch_binding(run)
    assert len(made) == 2
    os.remove(b.TORCH_STAMP)                       # a binding of unknown origin
    b.build_torch_binding(run)
    assert len(made) == 3


def test_binding_of_another_torch_is_refused(lib, monkeypatch):
    torch = pytest.importorskip("torch")
    if not os.path.exists(_lib.TORCH_BINDING_PATH):
        b.build()
    assert _lib.load_torch_binding().torch_version == torch.__version__
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    with pytest.raises(ImportError, match="built against"):
        _lib.load_torch_binding()


def test_headers_are_found_beside_an_nvcc_on_the_path(monkeypatch):
    if not os.path.exists("/usr/local/cuda/bin/nvcc"):
        pytest.skip("no nvcc in /usr/local/cuda")
    monkeypatch.setattr(b, "NVCC", "nvcc")
    monkeypatch.setenv("PATH", "/usr/local/cuda/bin" + os.pathsep + os.environ["PATH"])
    assert os.path.exists(os.path.join(b._cuda_root(), "include", "cuda_runtime.h"))
