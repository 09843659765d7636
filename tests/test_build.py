"""The build of the two compiled files: the library does not depend on the helper's."""
import pytest

from optimized_transducer_b200 import build


@pytest.fixture
def elsewhere(tmp_path, monkeypatch):
    """The helper's files in a folder of their own; the library is built already."""
    monkeypatch.setattr(build, "HELPER", str(tmp_path / "_tensors.so"))
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
