"""Runs the C++ test of the views that the attention operators refuse (tests/cpp/attention_refusals_test.cpp), without a device."""
import os
import subprocess


def test_cpp_attention_layer_refuses_views_that_do_not_fit(kd):
    import __graft_entry__ as ge
    exe = os.path.join(os.path.dirname(ge.build_cpp_dropin_test()), "attention_refusals_test")
    res = subprocess.run([exe], capture_output=True, text=True, timeout=300, env=dict(os.environ, CUDA_VISIBLE_DEVICES=""))
    assert res.returncode == 0, res.stdout + res.stderr
    assert "all checks passed" in res.stdout
