"""The normalisation kernels on the CPU, their buffers between pages that fault (cpu_kernels/norm_bounds.cpp): no
access out of range, no barrier that a thread misses, no result left unwritten.  At these sizes a workgroup visits one
block of a sample; test_norm_two_pass.py has those where it walks over several, and compares values."""
import os
import subprocess

import pytest

from deep_prob_feature_track_amd import build as B

HERE = os.path.dirname(os.path.abspath(__file__))
CLANG = os.path.join(B.LLVM_BIN, "clang++")
SIZES = [  # N, C, H, W, groups
    (1, 1, 1, 1, 1), (2, 6, 1, 1, 3), (1, 8, 5, 7, 2), (2, 13, 17, 5, 1), (2, 20, 9, 11, 4), (3, 30, 9, 11, 5), (1, 7, 3, 50, 7),
    (2, 96, 15, 20, 8), (2, 32, 33, 32, 8), (1, 257, 3, 5, 1), (2, 1030, 2, 3, 5), (1, 2056, 1, 3, 8), (2, 258, 5, 6, 129),
    (1, 400, 9, 7, 200), (1, 4, 100, 101, 1), (2, 128, 6, 8, 8), (1, 36, 20, 21, 3),
    (1, 260, 5, 7, 5)]


@pytest.fixture(scope="module")
def binary(tmp_path_factory):
    if not os.path.exists(CLANG):
        pytest.skip("no clang++ that knows vector types and 16-bit floats")
    out = str(tmp_path_factory.mktemp("cpu_kernels") / "norm_bounds")
    subprocess.run([CLANG, "-x", "c++", "-std=c++17", "-O1", "-w", f"-I{HERE}/cpu_kernels", f"-I{B.INC}", f"-I{B.CSRC}",
                    os.path.join(HERE, "cpu_kernels", "norm_bounds.cpp"), "-o", out], check=True)
    return out


@pytest.mark.parametrize("sizes", SIZES)
def test_kernels_stay_in_their_buffers(binary, sizes):
    r = subprocess.run([binary], input=" ".join(map(str, sizes)), capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr
    assert r.stdout == "6\n"
