"""GPU: what the prompts' attention kernels leave where a bounded wait ran out
(tests/cpp/test_kv4_timeout.cu; marks are set from the host, no kernel's wait runs out)."""

import os
import subprocess

import pytest

from conftest import PKG

pytestmark = pytest.mark.gpu


def test_marked_rows_are_not_written(cuda):
    exe = os.path.join(PKG, "build", "test_kv4_timeout")
    assert os.path.exists(exe), "build with make -C hrm-text-cuda_b200"
    res = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "all timeout tests passed" in res.stdout
