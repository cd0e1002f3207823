"""Compiles tests/native/muon_plan_test.cpp against csrc/muon_plan.hpp with the host compiler and its address sanitizer and runs it: the
order in which the products of orthogonalised momentum are launched, checked on the CPU."""
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host C++ compiler")
def test_every_operation_once_and_nothing_behind_a_list(tmp_path):
    exe = str(tmp_path / "muon_plan_test")
    subprocess.run(["g++", "-std=c++17", "-O1", "-g", "-Wall", "-fsanitize=address,undefined", "-fno-sanitize-recover=all",
                    "-I", os.path.join(ROOT, "polarai-framework_b200", "csrc"), "-o", exe,
                    os.path.join(ROOT, "tests", "native", "muon_plan_test.cpp")], check=True)
    out = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0, out.stdout + out.stderr
    assert " 0 failures" in out.stdout
