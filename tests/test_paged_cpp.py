"""The paged K/V cache's C++ structs (aurora_amd/csrc/aurora.hpp), compiled with g++ and linked against
libaurora_hip.so (tests/cpp/paged_check.cpp)."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
BIN = ROOT / "tests" / "cpp" / "paged_check"


def compile_paged_check(out: Path) -> None:
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-o", str(out), str(BIN) + ".cpp", f"-I{ROOT / 'include'}",
           f"-L{ROOT / 'aurora_amd'}", "-laurora_hip", f"-Wl,-rpath,{ROOT / 'aurora_amd'}",
           "-Wl,-rpath,$ORIGIN/../../aurora_amd", "-Wl,-rpath,/opt/rocm/lib"]
    subprocess.run(cmd, check=True, capture_output=True, text=True)


def test_paged_structs_build_and_refuse(tmp_path):
    exe = tmp_path / "paged_check"
    compile_paged_check(exe)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0 and "OK no-gpu" in res.stdout, res.stdout + res.stderr


@pytest.mark.gpu
def test_paged_structs_on_gpu():
    assert BIN.exists(), f"{BIN} is missing: __graft_entry__.build() compiles it"
    res = subprocess.run([str(BIN), "gpu"], capture_output=True, text=True, timeout=120)
    print(res.stdout, flush=True)
    assert res.returncode == 0 and "OK gpu" in res.stdout, res.stdout + res.stderr
