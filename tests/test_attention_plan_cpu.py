"""The preparation of the rotary plans with stand-ins for the CUDA runtime (tests/native/attention_plan_check.cu), on the CPU."""
import importlib
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def test_prepare_is_ordered_at_both_ends(tmp_path):
    """Frequencies of any device are read behind that device's work, and what prepare copies is there when it returns."""
    if not shutil.which("nvcc"):
        pytest.skip("needs nvcc")
    csrc = Path(importlib.import_module("deep-learning-math-kernel-research_b200").__file__).parent / "csrc"
    exe = tmp_path / "attention_plan_check"
    subprocess.check_call(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", "-cudart", "none", f"-I{csrc}", "-o", str(exe),
                           str(ROOT / "tests" / "native" / "attention_plan_check.cu"), str(csrc / "attention_api.cu")])
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stdout[-2000:]
