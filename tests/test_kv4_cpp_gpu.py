"""GPU: the C++ host layer's 4-bit cache methods (tests/cpp/test_kv4_ops.cpp): a
serving loop of prompt, eviction and single tokens against plain attention in double
precision over the cache's values, an update in place, and the refusals."""

import os
import subprocess

import pytest

from conftest import PKG

pytestmark = pytest.mark.gpu


def test_cpp_kv4():
    exe = os.path.join(PKG, "build", "test_kv4_ops")
    assert os.path.exists(exe), "build with make -C hrm-text-cuda_b200"
    res = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    print(res.stdout)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "all kv4 tests passed" in res.stdout
