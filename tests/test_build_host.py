"""The build of the torch binding around what a machine may lack: torch, its CUDA
part or a compiler, and its rebuild when torch or Python is another one."""
import importlib.util
import os
import subprocess
import sys
import types

import pytest

from __graft_entry__ import PKG_DIR, _load_build_script, load_package


@pytest.fixture
def script(tmp_path, monkeypatch):
    """build.py with its files in a folder of its own, a torch with a CUDA part and a
    compiler that writes the output and counts its calls."""
    b = _load_build_script()
    torch = tmp_path / "torch"
    (torch / "lib").mkdir(parents=True)
    (torch / "lib" / "libtorch_cuda.so").write_text("")
    (torch / "version.py").write_text("__version__ = '9.1'\n")
    for name in ("BINDING", "BINDING_STAMP"):
        monkeypatch.setattr(b, name, str(tmp_path / os.path.basename(getattr(b, name))))
    monkeypatch.setattr(b, "HERE", str(tmp_path / "package"))
    (tmp_path / "include").mkdir()
    (tmp_path / "include" / "nemo_relpos.h").write_text("")
    spec = types.SimpleNamespace(origin=str(torch / "__init__.py"))
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: spec)
    monkeypatch.setattr(b.shutil, "which", lambda name: "/usr/bin/" + name)
    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        open(b.BINDING, "w").close()
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    monkeypatch.setattr(subprocess, "run", run)
    return types.SimpleNamespace(b=b, torch=torch, calls=calls, spec=spec)


def test_binding_is_left_out_without_its_parts(script, monkeypatch):
    b = script.b
    (script.torch / "lib" / "libtorch_cuda.so").unlink()
    assert "CUDA part" in b._build_binding(False)
    (script.torch / "lib" / "libtorch_cuda.so").write_text("")
    with monkeypatch.context() as m:
        m.setattr(b.shutil, "which", lambda name: None)
        assert "g++" in b._build_binding(False)
    with monkeypatch.context() as m:
        m.setattr(importlib.util, "find_spec", lambda name: None)
        assert "not installed" in b._build_binding(True)
    assert not script.calls


def test_binding_follows_torch_and_python(script, monkeypatch):
    b = script.b
    b._build_binding(False)
    b._build_binding(False)
    assert len(script.calls) == 1  # nothing changed
    (script.torch / "version.py").write_text("__version__ = '9.2'\n")
    b._build_binding(False)
    b._build_binding(False)
    assert len(script.calls) == 2
    monkeypatch.setattr(sys, "version", "4.0")
    b._build_binding(False)
    assert len(script.calls) == 3
    b._build_binding(True)
    assert len(script.calls) == 4


def test_a_missing_binding_names_the_build_command(monkeypatch):
    _load_build_script().build()
    nrp = load_package()
    name = nrp.__name__ + "._nrp_torch"
    monkeypatch.setitem(sys.modules, name, None)  # an import of it fails
    monkeypatch.delattr(nrp, "_nrp_torch", raising=False)
    monkeypatch.delitem(sys.modules, nrp.__name__ + ".fp8", raising=False)
    spec = importlib.util.spec_from_file_location(nrp.__name__ + ".fp8",
                                                  os.path.join(PKG_DIR, "fp8.py"))
    with pytest.raises(nrp.NrpError, match="build.py"):
        spec.loader.exec_module(importlib.util.module_from_spec(spec))
