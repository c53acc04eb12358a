"""The extension module that calls DIOPI functions from Python: which library is taken."""
import importlib.machinery

import pytest


def test_libraries_of_other_interpreters_are_left_alone(diopi, tmp_path):
    (tmp_path / "dipu_b200_call.cpython-27-x86_64-linux-gnu.so").write_bytes(b"another interpreter's")
    assert diopi._load_call(str(tmp_path)) is None


def test_a_library_that_cannot_be_loaded_is_reported_and_left_out(diopi, tmp_path):
    """Built against another torch, say: the calls go through ctypes then."""
    (tmp_path / ("dipu_b200_call" + importlib.machinery.EXTENSION_SUFFIXES[0])).write_bytes(b"no library")
    with pytest.warns(RuntimeWarning, match="dipu_b200_call"):
        assert diopi._load_call(str(tmp_path)) is None


def test_no_library(diopi, tmp_path):
    assert diopi._load_call(str(tmp_path)) is None
