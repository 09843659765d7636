"""The build of the two compiled files: the library does not depend on the helper's."""
import os
import sys
import types

import pytest

from optimized_transducer_b200 import _lib, build


@pytest.fixture
def elsewhere(tmp_path, monkeypatch):
    """The helper's files in a folder of their own; the library is built already."""
    monkeypatch.setattr(build, "HELPER", str(tmp_path / "_tensors.so"))
    monkeypatch.setattr(build, "HELPER_STAMP", str(tmp_path / "_tensors.built"), raising=False)
    monkeypatch.setattr(build, "build_library", lambda force=False, verbose=False: build.LIB)
    return tmp_path


def test_the_library_is_there_without_the_helper(elsewhere, monkeypatch):
    broken = elsewhere / "tensors.cc"
    broken.write_text('#include "no_such_header.h"\n')
    monkeypatch.setattr(build, "HELPER_SOURCE", str(broken))
    (elsewhere / "_tensors.so").write_text("an older one")
    with pytest.warns(RuntimeWarning, match="_tensors.so was not built"):
        assert build.build() == build.LIB
    assert not (elsewhere / "_tensors.so").exists()          # nothing stale is left to be loaded


def test_no_compiler_and_no_torch(elsewhere, monkeypatch):
    for error in (FileNotFoundError("g++"), ImportError("torch")):
        def fail(error=error):
            raise error
        monkeypatch.setattr(build, "start_helper", fail)
        with pytest.warns(RuntimeWarning, match="_tensors.so was not built"):
            assert build.build() == build.LIB


def test_a_failed_library_still_fails(elsewhere, monkeypatch):
    def fail(force=False, verbose=False):
        raise RuntimeError("nvcc failed")
    monkeypatch.setattr(build, "build_library", fail)
    monkeypatch.setattr(build, "start_helper", lambda: None)
    with pytest.raises(RuntimeError, match="nvcc failed"):
        build.build()


def test_the_helper_is_built_again_for_another_torch(elsewhere, monkeypatch):
    started = []
    monkeypatch.setattr(build, "start_helper", lambda: started.append(1))
    for name, text in (("_tensors.so", ""), ("_tensors.built", build.built_for())):
        (elsewhere / name).write_text(text)
        later = os.path.getmtime(build.HELPER_SOURCE) + 10
        os.utime(elsewhere / name, (later, later))
    assert build.build() == build.LIB and not started
    (elsewhere / "_tensors.built").write_text("torch 1.0, Python 3.8")
    assert build.build() == build.LIB and started == [1]


def test_a_helper_for_another_torch_is_not_used(monkeypatch):
    monkeypatch.setattr(_lib, "_helper", None)
    assert _lib.tensors().built_for == build.built_for()
    monkeypatch.setattr(_lib, "_helper", None)
    other = types.ModuleType("optimized_transducer_b200._tensors")
    other.built_for = "torch 1.0, Python 3.8"
    monkeypatch.setitem(sys.modules, "optimized_transducer_b200._tensors", other)
    import optimized_transducer_b200
    monkeypatch.setattr(optimized_transducer_b200, "_tensors", other, raising=False)
    with pytest.raises(ImportError, match="built for torch 1.0"):
        _lib.tensors()
