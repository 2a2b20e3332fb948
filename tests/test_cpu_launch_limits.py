"""The host check of kvmem_hip_attention's launch size, without a GPU
(tests/operator_launch_limits.cpp)."""
from __future__ import annotations

import os
import subprocess

import pytest

from conftest import ROOT
from test_cpu_operator_refusals import HIPCC, build


def test_launches_that_do_not_fit_are_refused(tmp_path):
    if not os.path.exists(HIPCC):
        pytest.skip("hipcc is not installed")
    r = subprocess.run([str(build(tmp_path, ROOT / "tests" / "operator_launch_limits.cpp"))], capture_output=True,
                       text=True, timeout=120)
    assert r.returncode == 0 and "all refused" in r.stdout, r.stdout + r.stderr
