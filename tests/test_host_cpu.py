"""The library's host code on a simulated HIP runtime (tests/hostsim/): device memory is the
host's, the kernels that keep lengths and pages run as plain C++, and single calls fail where a
test picks them -- what a GPU cannot be asked to do."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "hostsim")

TESTS = ["append_of_many_tokens", "checks_allocate_nothing", "creation_out_of_host_memory", "error_of_one_call", "failed_calls",
         "failed_undo", "lengths_are_read_under_the_lock", "prompt_workspace",
         "streams_that_sit_out"]


@pytest.fixture(scope="module")
def host_tests():
    if shutil.which("make") is None or not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("make or hipcc is not installed")
    exe = os.path.join(HERE, "_build", "host_tests")
    r = subprocess.run(["make", "-s", "-j8", "-C", HERE, exe], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stdout + r.stderr
    return exe


@pytest.mark.parametrize("name", TESTS)
def test_host(host_tests, name):
    r = subprocess.run([host_tests, name], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def test_every_host_test_is_listed(host_tests):
    r = subprocess.run([host_tests], capture_output=True, text=True, timeout=60)
    assert r.stdout.split() == sorted(TESTS)
