"""An extension that does not load leaves the serving operators on ctypes, and says so."""

import pytest

from gdn_b200 import _lib, build, serving


def test_an_extension_that_does_not_load_is_left_out(gdn_lib, tmp_path, monkeypatch):
    stale = tmp_path / "gdn_b200_torch-stale.so"
    stale.write_bytes(b"not a shared object")
    monkeypatch.setattr(build, "torch_lib_path", lambda: str(stale))
    with pytest.warns(RuntimeWarning, match="gdn_b200_torch-stale"):
        assert _lib.torch_calls() is None
    monkeypatch.setattr(serving, "_calls", None)
    with pytest.warns(RuntimeWarning, match="build"):
        assert serving._torch_calls() is serving._Nothing
    assert serving._calls is serving._Nothing               # asked once


def test_no_extension_is_no_warning(gdn_lib, tmp_path, monkeypatch, recwarn):
    monkeypatch.setattr(build, "torch_lib_path", lambda: str(tmp_path / "none.so"))
    assert _lib.torch_calls() is None and not recwarn.list
