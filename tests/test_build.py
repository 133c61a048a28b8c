"""The build recipe where torch's or Python's headers are missing (no GPU)."""

import sys
import sysconfig

import pytest

from wisp_b200 import build


@pytest.mark.parametrize("what", ["torch", "Python.h"])
def test_the_library_builds_without_what_only_the_binding_needs(built_lib, monkeypatch, tmp_path, what):
    if what == "torch":
        monkeypatch.setitem(sys.modules, "torch.utils.cpp_extension", None)
        monkeypatch.setitem(sys.modules, "torch", None)
    else:
        real = sysconfig.get_paths
        monkeypatch.setattr(sysconfig, "get_paths", lambda: dict(real(), include=str(tmp_path)))
    with pytest.warns(RuntimeWarning, match="without the torch binding.*" + what):
        assert build.build() == built_lib
    assert build.BINDING.exists()  # built from this source before: kept
    # one of another source would not match the library
    other = tmp_path / "_paged_torch.so"
    other.write_bytes(b"")
    other.with_suffix(".so.sha256").write_text("0 0")
    monkeypatch.setattr(build, "BINDING", other)
    with pytest.warns(RuntimeWarning, match=what):
        build.build()
    assert not other.exists()
