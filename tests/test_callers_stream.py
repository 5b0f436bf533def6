"""Handles on a stream of the caller's (frz_open_on): what they refuse before
any device is asked for. CPU only."""
import ctypes
import subprocess
import sys
from pathlib import Path

import pytest

import frizzle_amd as fz
from frizzle_amd import _lib

ROOT = Path(__file__).resolve().parent.parent


def test_no_place_for_the_handle_refused():
    assert fz.load().frz_open_on(0, None, None, None) == 1
    with pytest.raises(fz.FrzError, match="frz_open_on: null out"):
        _lib.check(1)


def test_a_stream_a_thread_refused():
    handle = ctypes.c_void_p(1)
    status = fz.load().frz_open_on(0, 2, ctypes.byref(handle), None)  # hipStreamPerThread
    assert status == 1 and handle.value is None
    with pytest.raises(fz.FrzError, match="stream a thread"):
        _lib.check(status)


def test_a_stream_of_another_runtime_refused():
    # The library first, then torch, which loads a HIP runtime of its own.
    code = """
import frizzle_amd as fz
fz.load()
import torch
if len(fz.runtime._hip_runtimes()) < 2:
    print("one runtime")
else:
    try:
        fz.Device(0, stream=0)
    except fz.FrzError as e:
        print(e)
"""
    out = subprocess.run([sys.executable, "-c", code], cwd=ROOT, check=True, capture_output=True,
                         text=True).stdout
    if "one runtime" in out:
        pytest.skip("torch shares the library's runtime here")
    assert "two HIP runtimes" in out
