"""The build's parts: the C library does not depend on the autograd module over it. Stub compilers; nothing is
compiled and the built files are not touched."""
import os
import stat

import pytest

from lazylora_amd import build as b


@pytest.fixture
def stubs(tmp_path, monkeypatch):
    """Compilers that write the file after -o, the host one failing when told to; all outputs in tmp_path."""
    def script(name, text):
        path = tmp_path / name
        path.write_text("#!/bin/sh\n" + text)
        path.chmod(path.stat().st_mode | stat.S_IXUSR)
        return str(path)

    touch = 'while [ $# -gt 0 ]; do if [ "$1" = -o ]; then echo built > "$2"; fi; shift; done\n'
    monkeypatch.setattr(b, "HIPCC", script("hipcc", touch))
    monkeypatch.setenv("CXX", script("cxx", 'if [ -e "$0.fails" ]; then echo no Python.h >&2; exit 1; fi\n' + touch))
    monkeypatch.setattr(b, "HERE", str(tmp_path))
    monkeypatch.setattr(b, "LIB", str(tmp_path / "lib.so"))
    return tmp_path


def test_both_parts(stubs):
    assert b.build() == b.LIB
    assert os.path.exists(b.LIB) and list(stubs.glob(b.AUTOGRAD + "*.so"))


def test_library_without_the_autograd_module(stubs):
    """Where the module does not compile (no torch headers, no Python.h, no host compiler) the library is
    linked all the same, and the error says what failed."""
    (stubs / "cxx.fails").touch()
    with pytest.raises(RuntimeError, match="no Python.h"):
        b.build()
    assert os.path.exists(b.LIB) and not list(stubs.glob(b.AUTOGRAD + "*.so"))


def test_library_without_torch(stubs, monkeypatch):
    def no_torch(objdir):
        raise ImportError("No module named 'torch'")

    monkeypatch.setattr(b, "_autograd_commands", no_torch)
    with pytest.raises(RuntimeError, match="(?s)autograd module.*torch"):
        b.build()
    assert os.path.exists(b.LIB)


def test_host_compiler_absent(stubs, monkeypatch):
    monkeypatch.setenv("CXX", str(stubs / "nowhere"))
    with pytest.raises(RuntimeError, match="autograd module"):
        b.build()
    assert os.path.exists(b.LIB)


def test_library_that_does_not_compile(stubs):
    (stubs / "hipcc").write_text("#!/bin/sh\necho bad kernel >&2; exit 1\n")
    with pytest.raises(RuntimeError, match="bad kernel"):
        b.build()
    assert not os.path.exists(b.LIB)
