"""The extension module that calls DIOPI functions from Python: which library it takes, and what it accepts as an integer."""
import importlib.machinery

import numpy as np
import pytest
import torch


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


def _call_with(diopi, position):
    """A call that the library refuses for its shapes, before any device work."""
    t = [torch.zeros(2, 2) for _ in range(6)]
    diopi.diopiB200RopeAppendKV(diopi.Context(), *t, position)


@pytest.mark.parametrize("value", [1.5, "1", None, torch.tensor(1.5)])
def test_integers_are_not_made_from_other_things(diopi, value):
    with pytest.raises((TypeError, ValueError)):
        _call_with(diopi, value)


@pytest.mark.parametrize("value", [1, np.int64(1), True, torch.tensor(1)])
def test_integers_of_every_kind(diopi, value):
    """They reach the library."""
    with pytest.raises(diopi.DiopiError, match="q_out"):
        _call_with(diopi, value)
