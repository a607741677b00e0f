"""The library is built where the extension module of piton_b200.decode cannot be; no GPU needed."""

import shutil

import pytest

from piton_b200 import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A source tree of one small kernel."""
    if not shutil.which("nvcc"):
        pytest.skip("no nvcc")
    (tmp_path / "csrc").mkdir()
    (tmp_path / "csrc" / "one.cu").write_text('extern "C" __attribute__((visibility("default"))) int one() { return 1; }\n')
    for name, path in (("CSRC", "csrc"), ("OBJ", "obj"), ("LIB", "lib.so"), ("CALLS", "calls.so")):
        monkeypatch.setattr(build, name, str(tmp_path / path))
    return tmp_path


@pytest.mark.parametrize("error", [ImportError("no torch here"), RuntimeError("g++ failed"), FileNotFoundError("g++")])
def test_the_library_does_not_need_the_extension(tree, monkeypatch, error):
    def fails(verbose):
        raise error

    monkeypatch.setattr(build, "_build_calls", fails)
    (tree / "calls.so").write_text("of an earlier build")
    with pytest.warns(UserWarning, match="decode cannot be used"):
        assert build.build() == str(tree / "lib.so")
    assert (tree / "lib.so").exists() and not (tree / "calls.so").exists()


def test_a_compiler_without_torch_headers(tree, monkeypatch):
    # the real step with a host compiler that refuses the source
    monkeypatch.setenv("CXX", "false")
    (tree / "csrc" / "decode_calls.cpp").write_text("")
    with pytest.warns(UserWarning, match="calls.so was not built"):
        build.build()
    assert (tree / "lib.so").exists() and not (tree / "calls.so").exists()
