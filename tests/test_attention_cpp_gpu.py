"""Runs the C++ test of the attention operators (tests/cpp/attention_test.cpp) on the GPU."""
import os
import subprocess

import pytest

pytestmark = pytest.mark.gpu


def test_cpp_attention_layer(kd):
    import __graft_entry__ as ge
    exe = os.path.join(os.path.dirname(ge.build_cpp_dropin_test()), "attention_test")
    res = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "all checks passed" in res.stdout
