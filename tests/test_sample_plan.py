"""Where sampling finds a place among its histogram's steps
(qwenscriber_amd/csrc/sample_plan.h) on the CPU:
qwenscriber_amd/sanitize/sample_check.cpp, built with g++ and its sanitizers
(Makefile `sample_check`, no device code), asks for every running sum of
histograms added as a workgroup adds them, and for the numbers next to it. Such
sums fall, and rise over steps without tokens, by their last bits; the step
that is found has tokens all the same."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CHECK = os.path.join(ROOT, "qwenscriber_amd", "build", "sample_check")


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host C++ compiler")
def test_a_place_s_step_has_tokens():
    subprocess.run(["make", "-s", "-C", os.path.join(ROOT, "qwenscriber_amd"), "sample_check"], check=True)
    run = subprocess.run([CHECK], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout[-3000:] + run.stderr[-2000:]
    assert " 0 failures" in run.stdout, run.stdout
