"""A length of scale blocks that no call takes is refused before pools are allocated, in Python and in C++."""
import subprocess
from pathlib import Path

import pytest

from aurora_amd.gpu import PagedKvCache

ROOT = Path(__file__).resolve().parents[1]


class Nothing:
    def call(self, *args):
        raise AssertionError(args)


@pytest.mark.parametrize("page,block", [(256, 256), (512, 256), (16, 32), (16, 12), (16, 0)])
def test_python_refuses(page, block):
    with pytest.raises(ValueError, match=f"scale_len {block}"):
        PagedKvCache.zeros(Nothing(), 4, page, 2, 32, "e4m3", block)
    with pytest.raises(ValueError, match=f"scale_len {block}"):
        PagedKvCache(0x10000, 0x10000, 4, page, 2, 32, "e4m3", 0x10000, 0x10000, block)


def test_the_longest_is_taken():
    assert PagedKvCache(0x10000, 0x10000, 4, 256, 2, 32, "e4m3", 0x10000, 0x10000, 128).scales == 16


def test_cpp_refuses(tmp_path):
    exe = tmp_path / "lengths"
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-o", str(exe), str(ROOT / "tests" / "cpp" / "e4m3_lengths.cpp"),
                    f"-I{ROOT / 'include'}", f"-L{ROOT / 'aurora_amd'}", "-laurora_hip", f"-Wl,-rpath,{ROOT / 'aurora_amd'}",
                    "-Wl,-rpath,/opt/rocm/lib"], check=True, capture_output=True, text=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert res.returncode == 0, res.stdout + res.stderr
