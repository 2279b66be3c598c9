"""What the build compiles and when, on a package of one small source each."""
import os
import shutil

import pytest

from cgnet_b200 import build as b


@pytest.fixture
def package(tmp_path, monkeypatch):
    csrc = tmp_path / "csrc"
    csrc.mkdir()
    (csrc / "one.cu").write_text('extern "C" int one() { return 1; }\n')
    (csrc / b.BINDING_SOURCE).write_text('extern "C" int one();\nextern "C" int two() { return 2 * one(); }\n')
    header = tmp_path / "header.h"
    header.write_text("")
    for name, value in (("HERE", str(tmp_path)), ("CSRC", str(csrc)), ("SOURCES", ["one.cu"]), ("HEADER", str(header)), ("LIB", str(tmp_path / "libone.so")),
                        ("BINDING", str(tmp_path / "_two.so")), ("BINDING_TORCH", str(tmp_path / "_two.torch"))):
        monkeypatch.setattr(b, name, value)
    if shutil.which("g++") is None or not os.path.exists(b._nvcc()):
        pytest.skip("no compilers")
    return tmp_path


def test_a_binding_that_does_not_compile_leaves_the_library(package):
    (package / "csrc" / b.BINDING_SOURCE).write_text("#error no\n")
    with pytest.raises(RuntimeError, match=b.BINDING_SOURCE):
        b.build()
    assert os.path.exists(b.LIB) and not os.path.exists(b.BINDING) and b.needs_build()


def test_a_host_without_torch_gets_the_library(package, monkeypatch):
    monkeypatch.setattr(b, "_torch_version", lambda: None)
    assert b.build() == b.LIB and os.path.exists(b.LIB) and not os.path.exists(b.BINDING) and not b.needs_build()


def test_another_torch_rebuilds_the_binding_alone(package, monkeypatch):
    b.build()
    assert not b.needs_build()
    monkeypatch.setattr(b, "_torch_version", lambda: "1.0")
    assert b.needs_build()
    times = [os.path.getmtime(p) for p in (b.LIB, b.BINDING)]
    os.utime(b.BINDING, (times[1] + 1, times[1] + 1))
    b.build()
    assert not b.needs_build() and os.path.getmtime(b.LIB) == times[0] and open(b.BINDING_TORCH).read() == "1.0"


def test_sources_that_change_are_built_again(package):
    b.build()
    later = os.path.getmtime(b.BINDING) + 5
    for path, library in ((package / "csrc" / "one.cu", True), (package / "csrc" / b.BINDING_SOURCE, False)):
        os.utime(path, (later, later))
        assert b.needs_build() and b._library_stale() == library
        os.utime(b.LIB if library else b.BINDING, (later, later))
        assert not b.needs_build()
