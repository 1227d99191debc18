"""The host side of the language-model operators, without a GPU."""
import importlib.machinery
import importlib.util
import os
import subprocess
import sys

import pytest

from pdefa_b200 import build, lm

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

FAKE = """
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
import pdefa_b200 as pb

with FakeTensorMode():
    f = lambda *s: torch.empty(s, device="cuda")                              # noqa: E731
    q = lambda *s: torch.empty(s, device="cuda", dtype=torch.float8_e4m3fn)     # noqa: E731
    i = lambda *s: torch.empty(s, device="cuda", dtype=torch.int32)           # noqa: E731
    for call in (lambda: pb.ops_rms_norm(f(2, 8), f(8)), lambda: pb.ops_rms_norm(f(2, 8), f(8), residual=f(2, 8)),
                 lambda: pb.ops_rms_norm_fp8(f(2, 8), f(8)), lambda: pb.ops_matmul_fp8(q(2, 8), f(2, 1), q(4, 8), f(1, 1)),
                 lambda: pb.ops_matmul_grouped_fp8(q(2, 8), f(2, 1), q(3, 4, 8), f(3, 1, 1), i(4)),
                 lambda: pb.ops_sample(f(2, 8), f(2, 8)), lambda: pb.ops_sample(f(2, 8), f(2, 8), temperature=f(2))):
        try:
            call()
        except RuntimeError as e:
            print("refused")
"""


def test_tensors_without_storage_are_refused():
    """Fake CUDA tensors, as tracing makes them: an exception, not the interpreter's end."""
    pytest.importorskip("torch")
    r = subprocess.run([sys.executable, "-c", FAKE], cwd=ROOT, capture_output=True, text=True, timeout=300,
                       env={**os.environ, "PYTHONPATH": ROOT})
    assert r.returncode == 0, r.stderr[-2000:]
    assert r.stdout.split() == ["refused"] * 7


@pytest.fixture
def odd_torch(tmp_path, monkeypatch):
    """What build() sees as the installed torch: a package with CUDA but without headers; outputs go to tmp_path."""
    (tmp_path / "torch" / "lib").mkdir(parents=True)
    (tmp_path / "torch" / "__init__.py").write_text("")
    (tmp_path / "torch" / "version.py").write_text("__version__ = '0.0.1+none'\n")
    (tmp_path / "torch" / "lib" / "libc10_cuda.so").write_text("")
    find = importlib.util.find_spec
    spec = importlib.machinery.ModuleSpec("torch", None, origin=str(tmp_path / "torch" / "__init__.py"))
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: spec if name == "torch" else find(name, *a))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "libpdefa_native.so"))
    monkeypatch.setattr(build, "LIB_DIR", str(tmp_path))
    return tmp_path


def test_engine_builds_without_the_binding(odd_torch):
    with pytest.warns(RuntimeWarning, match="no binding for torch"):
        assert build.build() == str(odd_torch / "libpdefa_native.so")
    assert (odd_torch / "libpdefa_native.so").stat().st_size > 1000000
    assert not list(odd_torch.glob("lm_torch*.so"))


def test_engine_builds_without_a_compiler_for_the_binding(odd_torch, monkeypatch):
    run = subprocess.run

    def no_gxx(cmd, **kw):
        if cmd[0] == "g++":
            raise FileNotFoundError("g++")
        return run(cmd, **kw)

    monkeypatch.setattr(subprocess, "run", no_gxx)
    with pytest.warns(RuntimeWarning, match="g\\+\\+"):
        assert os.path.exists(build.build())


def test_torch_without_cuda_has_no_binding(odd_torch, monkeypatch, recwarn):
    pytest.importorskip("torch")
    (odd_torch / "torch" / "lib" / "libc10_cuda.so").unlink()
    assert os.path.exists(build.build()) and not recwarn.list
    monkeypatch.setattr(lm, "_B", None)
    with pytest.raises(TypeError, match="no CUDA"):
        lm.ops_sample(None, None)


def test_first_call_says_why_there_is_no_binding(odd_torch, monkeypatch):
    pytest.importorskip("torch")
    monkeypatch.setattr(lm, "_B", None)
    with pytest.raises(RuntimeError, match="torch binding failed"):
        lm.ops_sample(None, None)


def test_binding_is_of_the_installed_versions(odd_torch, monkeypatch):
    """One that was built for another torch or Python is not taken, however new it is."""
    pytest.importorskip("torch")
    root = str(odd_torch / "torch")
    first = build.torch_lib(root)
    open(first, "w").close()
    (odd_torch / "torch" / "version.py").write_text("__version__ = '0.0.2'\ndebug = False\n")
    second = build.torch_lib(root)
    monkeypatch.setattr(sys.implementation, "cache_tag", "cpython-399")
    assert len({first, second, build.torch_lib(root)}) == 3
    monkeypatch.setattr(lm, "_B", None)
    with pytest.raises(RuntimeError, match="torch binding failed"):      # it is built, not loaded
        lm.ops_sample(None, None)


def test_loaded_binding_is_the_installed_versions_own():
    torch = pytest.importorskip("torch")
    with pytest.raises(TypeError):
        lm.ops_sample(None, None)
    assert torch.__version__ in lm._B.__spec__.loader.path and sys.implementation.cache_tag in lm._B.__spec__.loader.path
