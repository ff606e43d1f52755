"""How group norm cuts views up, checked on the host: ``norm_plan_check.cu`` runs the planning code of
the kernels' header over many sizes."""

import shutil
import subprocess
from pathlib import Path

import pytest

from diffrast_b200 import build

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("nvcc") is None and not Path("/usr/local/cuda/bin/nvcc").exists(),
                    reason="needs nvcc")
def test_plans_bound_the_rows_of_a_thread(tmp_path):
    exe = tmp_path / "norm_plan_check"
    subprocess.run([build.nvcc(), *build.ARCH, *build.FLAGS, f"-I{build.CSRC}",
                    str(ROOT / "tests" / "norm_plan_check.cu"), "-o", str(exe)],
                   check=True, capture_output=True, text=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout
    assert int(out.stdout.split()[0]) > 100000
