"""GPU: the C++ layer's attention workspace outlives the graphs that were captured with
it (tests/cpp/test_kv4_workspace.cpp)."""

import os
import subprocess

import pytest

from conftest import PKG

pytestmark = pytest.mark.gpu


def test_captured_call_replays_after_the_workspace_grew(cuda):
    exe = os.path.join(PKG, "build", "test_kv4_workspace")
    assert os.path.exists(exe), "build with make -C hrm-text-cuda_b200"
    res = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "all workspace tests passed" in res.stdout
