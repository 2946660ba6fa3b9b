"""build.py: libfp4x.so, the C ABI's library, needs hipcc alone.  Compilers are
stand-ins that write their output file, or fail."""
import importlib.util
import os
import stat

import pytest

from conftest import PKG

TOOL = """#!/bin/sh
{fail}
while [ $# -gt 0 ]; do
  if [ "$1" = -o ]; then echo built > "$2"; fi
  shift
done
"""


def tool(path, fail=""):
    path.write_text(TOOL.format(fail=fail))
    path.chmod(path.stat().st_mode | stat.S_IXUSR)
    return str(path)


@pytest.fixture
def B(tmp_path, monkeypatch):
    """build.py with its outputs in a folder of the test's and a hipcc that succeeds."""
    spec = importlib.util.spec_from_file_location("fp4x_build_under_test", os.path.join(PKG, "build.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    hipcc = tool(tmp_path / "hipcc")
    monkeypatch.setattr(mod, "_hipcc", lambda: hipcc)
    for name, at in (("HERE", ""), ("OBJ", "_build"), ("LIB", "libfp4x.so"), ("HOST", "_fp4x_host.so")):
        monkeypatch.setattr(mod, name, str(tmp_path / at))
    return mod


def test_both_libraries(B, tmp_path, monkeypatch):
    monkeypatch.setenv("CXX", tool(tmp_path / "cxx"))
    assert B.build() == B.LIB
    assert os.path.exists(B.LIB) and os.path.exists(B.HOST)


def test_c_library_without_a_host_compiler(B, tmp_path, monkeypatch):
    for cxx, why in ((tool(tmp_path / "cxx", "echo no Python.h >&2; exit 1"), "no Python.h"),
                     (str(tmp_path / "absent"), "absent")):
        monkeypatch.setenv("CXX", cxx)
        with open(B.HOST, "w") as f:
            f.write("of an earlier build")
        with pytest.raises(RuntimeError, match=why):   # said, with the C library in place
            B.build()
        assert os.path.exists(B.LIB) and not os.path.exists(B.HOST)
        os.remove(B.LIB)


def test_c_library_without_torch(B, tmp_path, monkeypatch, capsys):
    find = importlib.util.find_spec
    monkeypatch.setenv("CXX", tool(tmp_path / "cxx"))
    monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    assert B.build() == B.LIB
    assert os.path.exists(B.LIB) and not os.path.exists(B.HOST)
    assert "torch" in capsys.readouterr().err


def test_kernels_that_do_not_compile(B, tmp_path, monkeypatch):
    monkeypatch.setenv("CXX", tool(tmp_path / "cxx"))
    hipcc = tool(tmp_path / "hipcc", "echo broken >&2; exit 1")
    monkeypatch.setattr(B, "_hipcc", lambda: hipcc)
    with pytest.raises(RuntimeError, match="broken"):
        B.build()
    assert not os.path.exists(B.LIB) and not os.path.exists(B.HOST)
