"""The switch that turns off overlapped launches in tuning builds reaches every one of them."""
import importlib
import os
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


def _csrc():
    return Path(importlib.import_module("deep-learning-math-kernel-research_b200").__file__).parent / "csrc"


def test_launches_ask_one_place_whether_they_overlap():
    said = {p.name: p.read_text().count("programmaticStreamSerializationAllowed") for p in _csrc().glob("*.cu*")}
    assert {name for name, n in said.items() if n} == {"elb_common.cuh"} and said["elb_common.cuh"] == 1


@pytest.mark.parametrize("tuning,env,want", [(True, "1", "0"), (True, "0", "1"), (True, None, "1"), (False, "1", "1")])
def test_the_switch(tmp_path, tuning, env, want):
    if not shutil.which("nvcc"):
        pytest.skip("needs nvcc")
    exe = tmp_path / "overlap_check"
    subprocess.check_call(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O0", f"-I{_csrc()}", "-o", str(exe),
                           str(ROOT / "tests" / "native" / "overlap_check.cu")] + (["-DELB_TUNING"] if tuning else []))
    full = {k: v for k, v in os.environ.items() if k != "ELB_NO_OVERLAP"}
    if env is not None:
        full["ELB_NO_OVERLAP"] = env
    assert subprocess.run([str(exe)], env=full, capture_output=True, text=True).stdout.strip() == want
