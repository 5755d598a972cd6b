"""Runs the C++ device test of what the host mirror's paged cache refuses (tests/host/test_host_paged_errors.cpp)."""
import os
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
BIN = os.path.join(HERE, "host", "test_host_paged_errors")


def test_binary_is_built_and_reports_a_missing_device():
    import torch
    assert os.path.exists(BIN), "run __graft_entry__.build() (make -C tests/host)"
    if torch.cuda.is_available():
        pytest.skip("device present")
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=60)
    assert r.returncode == 77 and "no HIP device" in r.stdout


@pytest.mark.gpu
def test_refusals_on_device():
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=120)
    print(r.stdout[-3000:], r.stderr[-2000:], flush=True)
    assert r.returncode == 0 and "ALL PASS" in r.stdout, r.stdout[-3000:]
