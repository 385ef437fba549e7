"""Building the attention operators' torch binding, without a GPU."""
import importlib.machinery
import importlib.util
import os

import pytest

from fusedkernellibrary_amd import build


@pytest.mark.parametrize("libraries", [None, ["libc10.so", "libtorch_cpu.so"], ["libc10.so", "libc10_cuda.so"]])
def test_without_a_torch_for_rocm_there_is_nothing_to_bind(tmp_path, monkeypatch, capsys, libraries):
    """No torch, one for the CPU, one for another make of GPU: the library's build goes on without the binding, whose file stays as it is."""
    spec = None
    if libraries is not None:
        (tmp_path / "lib").mkdir()
        for name in libraries:
            (tmp_path / "lib" / name).touch()
        spec = importlib.machinery.ModuleSpec("torch", None, is_package=True)
        spec.submodule_search_locations.append(str(tmp_path))
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: spec)
    monkeypatch.setenv("CXX", str(tmp_path / "no-compiler"))
    there = os.path.join(build.PKG, "_attention.so")
    before = os.path.getmtime(there) if os.path.exists(there) else None
    assert build.build_torch_binding() is None
    assert "no torch for ROCm" in capsys.readouterr().out
    assert before == (os.path.getmtime(there) if os.path.exists(there) else None)
