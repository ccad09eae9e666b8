"""Compiles the checks of the launch plans (tests/cpp/plan_checks.cpp): they are evaluated by the compiler."""
import subprocess
from pathlib import Path

from heterofusedkernels_b200 import build

ROOT = Path(__file__).resolve().parent.parent


def test_launch_plans():
    run = subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsyntax-only", f"-I{ROOT / 'heterofusedkernels_b200' / 'csrc'}",
                          f"-I{build._cuda_home() / 'include'}", str(ROOT / "tests" / "cpp" / "plan_checks.cpp")], capture_output=True, text=True)
    assert run.returncode == 0, run.stderr
