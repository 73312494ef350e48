"""The host side of the transformer operators with stand-ins for the CUDA runtime and the kernels (tests/native/op_plan_check.cu), on the CPU."""
import importlib
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parent.parent


@pytest.fixture(scope="module")
def check(tmp_path_factory):
    if not shutil.which("nvcc"):
        pytest.skip("needs nvcc")
    csrc = Path(importlib.import_module("deep-learning-math-kernel-research_b200").__file__).parent / "csrc"
    exe = tmp_path_factory.mktemp("op_plan") / "op_plan_check"
    subprocess.check_call(["nvcc", "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", "-cudart", "none", f"-I{csrc}", "-o", str(exe),
                           str(ROOT / "tests" / "native" / "op_plan_check.cu"), str(csrc / "op_api.cu")])

    def run(case):
        r = subprocess.run([str(exe), case], capture_output=True, text=True, timeout=60)
        assert r.returncode == 0 and r.stdout == "ok\n", r.stdout[-2000:]
    return run


def test_calls_on_several_streams_take_turns_in_the_workspace(check):
    check("streams")


def test_streams_that_share_a_handle_take_turns_in_the_workspace(check):
    """cudaStreamPerThread is one handle for a stream of each thread, and a destroyed stream's handle may come back."""
    check("one_handle")


def test_a_call_that_failed_half_way_is_waited_for(check):
    check("failed")


def test_experts_counts_start_from_zero_behind_failed_and_captured_calls(check):
    check("counts")


def test_weights_on_another_device_are_copied(check):
    check("devices")


def test_slots_up_to_the_most_of_a_plan_are_shared_out(check):
    check("shares")
