"""How the dense layers' host extension is built and found (no GPU)."""
import os
import shutil
import subprocess

import pytest

from vaayu_b200 import build, dense


@pytest.fixture
def fake_tree(tmp_path, monkeypatch):
    """The build's outputs under tmp_path, and a compiler that only writes its output file."""
    log, cxx = tmp_path / "calls", tmp_path / "cxx"
    cxx.write_text(f'#!/bin/sh\necho run >> {log}\nwhile [ $# -gt 0 ]; do [ "$1" = -o ] && echo x > "$2"; shift; done\n')
    cxx.chmod(0o755)
    monkeypatch.setenv("CXX", str(cxx))
    monkeypatch.setattr(build, "HOST_LIB", tmp_path / "_dense_host.so")
    monkeypatch.setattr(build, "OBJ", tmp_path / "_build")
    monkeypatch.setattr(build, "HOST_MADE", tmp_path / "_build" / "_dense_host.txt", raising=False)

    def compiles():
        before = len(log.read_text().split()) if log.exists() else 0
        build.build_host()
        return len(log.read_text().split()) - before

    return compiles


def test_the_extension_is_rebuilt_for_another_torch_or_python(fake_tree, monkeypatch):
    import platform

    import torch
    assert fake_tree() == 1
    assert fake_tree() == 0
    monkeypatch.setattr(torch, "__version__", "9.9.0")
    assert fake_tree() == 1 and fake_tree() == 0
    monkeypatch.setattr(platform, "python_version", lambda: "9.9.9")
    assert fake_tree() == 1 and fake_tree() == 0
    os.utime(build.HOST_LIB, (0, 0))                       # an older library than its source
    assert fake_tree() == 1 and fake_tree() == 0


def test_an_extension_that_does_not_load_names_the_cause(monkeypatch):
    import sys
    monkeypatch.setattr(dense, "_HOST", None)
    monkeypatch.setitem(sys.modules, "vaayu_b200._dense_host", None)      # import raises
    monkeypatch.delattr("vaayu_b200._dense_host", raising=False)
    with pytest.raises(RuntimeError, match="does not load .*vaayu_b200._dense_host"):
        dense._host()


@pytest.mark.skipif(not shutil.which("readelf"), reason="binutils not available")
def test_the_extension_uses_the_process_s_c_plus_plus_library():
    """A second C++ library inside the extension has streams of its own that nobody initialised: an error
    message with a number in it (every refused C call has one) ended the process."""
    out = subprocess.run(["readelf", "-d", str(build.HOST_LIB)], capture_output=True, text=True, check=True).stdout
    assert "libstdc++.so.6" in out
    symbols = subprocess.run(["readelf", "-W", "--dyn-syms", str(build.HOST_LIB)], capture_output=True, text=True,
                             check=True).stdout
    assert not [s for s in symbols.splitlines() if "_ZNSo9_M_insert" in s and " UND " not in s]
