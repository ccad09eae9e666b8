"""Compiles and runs the CPU-only checks of the kernels' bounded waits (tests/cpp/wait_checks.cpp), and looks where the prefix kernel
uses them: a failure path cannot be run on a GPU without making something fail there."""
import re
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parent.parent
CSRC = ROOT / "heterofusedkernels_b200" / "csrc"


def test_bounded_waits(tmp_path):
    exe = tmp_path / "wait_checks"
    build = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{CSRC}", str(ROOT / "tests" / "cpp" / "wait_checks.cpp"), "-o", str(exe)],
                           capture_output=True, text=True)
    assert build.returncode == 0, build.stdout + build.stderr
    run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0 and "wait checks ok" in run.stdout, run.stdout + run.stderr


def test_the_prefix_kernel_drains_its_products_before_it_frees_tensor_memory():
    text = (CSRC / "prefix_tensor.cuh").read_text()
    last_commit, free = text.rindex("tc_commit(&sm.o_full"), text.rindex("tcgen05.dealloc")
    between = text[last_commit:free]
    assert re.search(r"\bdrain\(", between) and "wait_warp(&sm.o_full" not in between
