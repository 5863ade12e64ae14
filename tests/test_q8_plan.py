"""Planning of the 8-bit layer's launches over whole ranges of sizes, without a GPU: tests/cpp/q8_plan.cpp
compiled against the library's own planning header."""
import os
import shutil
import subprocess

import pytest

from conftest import PKG_DIR, ROOT


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    cxx = shutil.which("g++")
    if not cxx:
        pytest.skip("no g++")
    exe = str(tmp_path_factory.mktemp("plan") / "q8_plan")
    res = subprocess.run([cxx, "-std=c++17", "-O2", "-I", os.path.join(PKG_DIR, "csrc"), "-o", exe,
                          os.path.join(ROOT, "tests", "cpp", "q8_plan.cpp")], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr
    return lambda *args: subprocess.run([exe, *args], capture_output=True, text=True, timeout=300)


def test_rings_fit_shared_memory(plan):
    run = plan("ring")
    assert run.returncode == 0 and run.stdout.startswith("ok"), run.stdout


def test_weight_gradient_sums_at_most_768_tokens_an_accumulator(plan):
    run = plan("parts")
    assert run.returncode == 0 and run.stdout.startswith("ok"), run.stdout


def test_aligning_copy_reads_inside_its_operand(plan):
    run = plan("words")
    assert run.returncode == 0 and run.stdout.startswith("ok"), run.stdout
