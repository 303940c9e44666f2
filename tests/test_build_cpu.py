"""The Python binding's extension is built for the torch that is there, and is not needed."""
import os
import sys

import pytest

pytest.importorskip("torch")

from openasr_b200 import build  # noqa: E402


@pytest.fixture
def ops(tmp_path, monkeypatch):
    """where the extension goes, and a compiler that notes its calls and writes what it was asked for"""
    out, log = tmp_path / "_torch_ops.so", tmp_path / "calls"
    cxx = tmp_path / "cxx"
    cxx.write_text(f"#!{sys.executable}\nimport sys\nopen({str(log)!r}, 'a').write('x')\nopen(sys.argv[sys.argv.index('-o') + 1], 'w')\n")
    cxx.chmod(0o755)
    log.write_text("")
    monkeypatch.setattr(build, "TORCH_OPS", str(out))
    monkeypatch.setattr(build, "HOST_CXX", str(cxx))
    return out, log


def test_an_extension_that_does_not_compile_is_left_out(ops, tmp_path, monkeypatch, capsys):
    """an older one is no stand-in; the binding's calls go through ctypes"""
    out, _ = ops
    out.write_text("of another day")
    os.utime(out, (1, 1))
    failing = tmp_path / "failing"
    failing.write_text("#!/bin/sh\necho no such header >&2\nexit 1\n")
    failing.chmod(0o755)
    monkeypatch.setattr(build, "HOST_CXX", str(failing))
    build._build_torch_ops()
    assert not out.exists() and "no such header" in capsys.readouterr().err


def test_the_extension_is_built_again_for_another_torch(ops, monkeypatch):
    out, log = ops
    build._build_torch_ops()
    build._build_torch_ops()
    assert out.exists() and log.read_text() == "x", "built once"
    monkeypatch.setattr(sys, "version", "another Python")
    build._build_torch_ops()
    assert log.read_text() == "xx"
    stamp = out.with_name(out.name + ".for")
    stamp.write_text(stamp.read_text().replace("__version__", "__version__ = 'another torch' #"))
    build._build_torch_ops()
    assert log.read_text() == "xxx"
    stamp.unlink()  # built by a version that kept no record
    build._build_torch_ops()
    assert log.read_text() == "xxxx" and stamp.exists()


def test_the_extension_goes_where_torchs_headers_have_gone(ops, monkeypatch):
    out, log = ops
    build._build_torch_ops()
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None)
    build._build_torch_ops()
    assert not out.exists() and log.read_text() == "x"
