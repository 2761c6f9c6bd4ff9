"""`__graft_entry__.build()` on a tree whose tests are others than this one's: it needs no test module,
and compiles the C++ checks that are there."""
import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]

# The libraries are built already, and are what the checks link against: only what follows them is run.
SCRIPT = """
import __graft_entry__, oracle
from aurora_amd import build
build.build = lambda verbose=False: None
oracle.build = lambda: None
__graft_entry__.build()
"""


@pytest.mark.parametrize("checks", [None, [], ["api_check.cpp"], ["api_check.cpp", "paged_check.cpp"]])
def test_build_takes_the_checks_that_are_there(tmp_path, checks):
    for name in ("aurora_amd", "oracle", "include"):
        (tmp_path / name).symlink_to(ROOT / name)
    shutil.copy(ROOT / "__graft_entry__.py", tmp_path)
    cpp = tmp_path / "tests" / "cpp"
    if checks is not None:
        cpp.mkdir(parents=True)
        (tmp_path / "tests" / "__init__.py").touch()
        for name in checks:
            shutil.copy(ROOT / "tests" / "cpp" / name, cpp)
    res = subprocess.run([sys.executable, "-c", SCRIPT], cwd=tmp_path, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0, res.stdout + res.stderr
    for name in checks or []:
        exe = cpp / name[:-len(".cpp")]
        assert exe.exists()
        if os.path.exists("/dev/kfd"):
            continue  # a GPU host: the gpu-marked tests run the checks
        run = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
        assert run.returncode == 0 and "OK no-gpu" in run.stdout, run.stdout + run.stderr


def test_a_check_that_does_not_compile_ends_the_build(tmp_path):
    for name in ("aurora_amd", "oracle", "include"):
        (tmp_path / name).symlink_to(ROOT / name)
    shutil.copy(ROOT / "__graft_entry__.py", tmp_path)
    cpp = tmp_path / "tests" / "cpp"
    cpp.mkdir(parents=True)
    (cpp / "odd_check.cpp").write_text("int main() { return no_such_name; }\n")
    res = subprocess.run([sys.executable, "-c", SCRIPT], cwd=tmp_path, capture_output=True, text=True, timeout=300)
    assert res.returncode != 0 and "odd_check" in res.stderr and "no_such_name" in res.stderr, res.stdout + res.stderr
