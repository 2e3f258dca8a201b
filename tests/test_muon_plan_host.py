"""The shares of tiles of the Newton-Schulz products, as the library's own code cuts and walks them
(arcqml_b200/csrc/muon_plan.h, compiled for the CPU by muon_plan_check.cpp)."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
CSRC = os.path.join(os.path.dirname(HERE), "arcqml_b200", "csrc")


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_every_step_is_taken_once(tmp_path):
    exe = str(tmp_path / "muon_plan_check")
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", CSRC,
                    os.path.join(HERE, "muon_plan_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
    plans, tiles, cut = map(int, r.stdout.split())
    assert plans == 6000 and tiles > 100_000 and cut > 1000
