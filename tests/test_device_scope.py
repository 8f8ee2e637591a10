"""The device that a call runs on, and the caller's current device behind it (csrc/device_scope.h),
without a GPU: the header's logic against a stand-in for CUDA, and the Python layer's question
whether a stream is being captured against a stand-in for torch's."""

import contextlib
import os
import shutil
import subprocess

import pytest
import torch

from conftest import PKG
from llm_kernels import _lib

HERE = os.path.dirname(os.path.abspath(__file__))


def test_calls_run_on_their_device_and_leave_the_callers(tmp_path):
    cxx = shutil.which("g++") or shutil.which("c++")
    if cxx is None:
        pytest.skip("no C++ compiler")
    exe = str(tmp_path / "device_scope")
    r = subprocess.run([cxx, "-std=c++17", "-Wall", "-Werror", "-I" + os.path.join(PKG, "csrc"), "-o", exe,
                        os.path.join(HERE, "device_scope.cpp")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout


def test_capture_is_asked_of_the_tensors_device(monkeypatch):
    """A capture on device 1's current stream counts for device 1's tensors, whichever device is current."""
    now = [0]

    @contextlib.contextmanager
    def device(index):
        before, now[0] = now[0], index
        yield
        now[0] = before

    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: now[0] == 1)
    assert _lib._capturing(1) is True and _lib._capturing(0) is False and now == [0]
    now[0] = 1
    assert _lib._capturing(1) is True and _lib._capturing(0) is False and now == [1]
