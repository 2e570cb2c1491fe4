"""The paged attention's plan for tables of any length (no GPU work)."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


def test_every_table_has_a_plan(tmp_path):
    """kv_split.cuh compiled for the host; a plan without a split ends the process by a division by zero."""
    nvcc = next((c for c in ("/usr/local/cuda/bin/nvcc", shutil.which("nvcc")) if c and Path(c).exists()), None)
    if nvcc is None:
        pytest.skip("nvcc not found")
    exe = tmp_path / "kv_plan_check"
    build = subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr",
                            "-I" + str(ROOT / "inferq_b200" / "csrc"), "-I" + str(ROOT / "include"),
                            str(ROOT / "tests" / "native" / "kv_plan_check.cu"), "-o", str(exe)],
                           capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, (run.returncode, run.stdout)
