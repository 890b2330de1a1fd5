"""What is asked of a device once: kept by device, and a failed query is not kept.  CPU only."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "lightship_b200", "csrc")


def test_counts_are_kept_by_device_and_failures_are_not(tmp_path):
    cc = shutil.which("g++") or shutil.which("c++")
    if cc is None:
        pytest.skip("no C++ compiler")
    exe = str(tmp_path / "device_count_check")
    subprocess.run([cc, "-O1", "-std=c++17", "-Wall", "-Werror", "-pthread", "-I", CSRC,
                    os.path.join(HERE, "device_count_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


def test_no_process_wide_answer_about_a_device():
    """The prompt attention's choice of a cluster size goes by the device it launches on, and a query that
    fails does not refuse the call."""
    with open(os.path.join(CSRC, "attention_prefill.cu")) as f:
        source = f.read()
    at = source.index("cudaOccupancyMaxActiveClusters")
    around = source[source.rindex("template <bool BF16", 0, at):at + 400]
    assert "DeviceCount" in around and "once_flag" not in around and "cuda_error" not in around
