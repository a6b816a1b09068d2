"""The paged cache through the C++ mirror (include/lumen_b200.hpp): compiles and links on the CPU, gives the right numbers on a GPU."""
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
LIBDIR = ROOT / "lumen_b200" / "lib"


@pytest.fixture(scope="module")
def binary(tmp_path_factory, L):
    out = tmp_path_factory.mktemp("pagedmirror") / "paged_mirror_check"
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-I", str(ROOT / "include"), str(ROOT / "tests" / "cpp" / "paged_mirror_check.cpp"),
                        "-L", str(LIBDIR), "-llumen_b200", f"-Wl,-rpath,{LIBDIR}", "-o", str(out)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-3000:]
    return out


def test_compiles_and_reports_a_missing_device(binary):
    import torch
    if torch.cuda.is_available():
        pytest.skip("covers the no-device path")
    r = subprocess.run([str(binary), "--no-gpu"], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "Error code=7" in r.stdout, r.stdout + r.stderr


@pytest.mark.gpu
def test_tokens_through_the_mirror(binary):
    r = subprocess.run([str(binary)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr
