"""What a training step's row operators launch at every size that their entry points
take, without a GPU: the check of tests/cpp/host_launch.cpp that names them, under
AddressSanitizer and UndefinedBehaviorSanitizer."""
import os
import subprocess

import pytest

from tests.test_host_launch import _binary


def test_row_operators(tmp_path):
    if subprocess.run(["g++", "--version"], capture_output=True).returncode != 0:
        pytest.skip("no g++")
    env = dict(os.environ)
    env["ASAN_OPTIONS"] = "detect_leaks=0:halt_on_error=1"
    env["UBSAN_OPTIONS"] = "halt_on_error=1:print_stacktrace=1"
    r = subprocess.run([_binary(), "row_operators"], capture_output=True, text=True, env=env, cwd=tmp_path, timeout=300)
    out = r.stdout + r.stderr
    assert "AddressSanitizer" not in out and "runtime error" not in out, out[-4000:]
    assert r.returncode == 0 and "row_operators ok" in r.stdout, out[-4000:]
