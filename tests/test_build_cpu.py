"""The build where a part of it cannot be had."""
import ctypes

import pytest

from compactlogic_amd import build


@pytest.fixture
def elsewhere(tmp_path, monkeypatch):
    """A build of one small source in a folder of its own, over what an earlier one left."""
    (tmp_path / "csrc").mkdir()
    (tmp_path / "csrc" / "one.hip").write_text('extern "C" int answer(void) { return 42; }\n')
    for name, path in [("CSRC", "csrc"), ("BUILD", "_build"), ("LIB", "libone.so"),
                       ("AUTOGRAD", "_one.so")]:
        monkeypatch.setattr(build, name, tmp_path / path)
    build.AUTOGRAD.write_bytes(b"of an earlier build")
    return build


def _no_compiler():
    raise RuntimeError("g++ not found")


def _no_torch():
    raise ImportError("no module named setuptools")


def _no_link(obj):
    raise RuntimeError("link of the autograd extension failed")


@pytest.mark.parametrize("what,how,message", [
    ("_compile_autograd", _no_compiler, "g\\+\\+ not found"),
    ("_compile_autograd", _no_torch, "setuptools"),
    ("_link_autograd", _no_link, "link of the autograd")])
def test_the_library_is_built_without_the_extension(elsewhere, monkeypatch, what, how, message):
    monkeypatch.setattr(elsewhere, "_compile_autograd", lambda: None)
    monkeypatch.setattr(elsewhere, "_link_autograd", lambda obj: None)
    monkeypatch.setattr(elsewhere, what, how)
    with pytest.raises(RuntimeError, match=message):
        elsewhere.build(verbose=False)
    assert ctypes.CDLL(str(elsewhere.LIB)).answer() == 42
    assert not elsewhere.AUTOGRAD.exists()


def test_no_library_without_the_kernels(elsewhere, monkeypatch):
    """A kernel that does not compile leaves the earlier build as it was."""
    monkeypatch.setattr(elsewhere, "_compile_autograd", lambda: None)
    (elsewhere.CSRC / "one.hip").write_text("this is no source\n")
    with pytest.raises(RuntimeError, match="hipcc failed on one.hip"):
        elsewhere.build(verbose=False)
    assert not elsewhere.LIB.exists()
    assert elsewhere.AUTOGRAD.read_bytes() == b"of an earlier build"
