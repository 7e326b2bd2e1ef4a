"""The square root that the 8-bit AdamW state is made with (csrc/pair_math.cuh) is the
rounded one for every fp32 number, so that codes and scales are those of a scalar
evaluation.  CPU: the program compiles for sm_100a.  GPU: it goes through all of them."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")


def _build(tmp_path):
    out = str(tmp_path / "root_all")
    subprocess.check_call([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-O3", "-std=c++17", "-diag-suppress", "177",
                           "-I", os.path.join(ROOT, "coconet_b200", "csrc"), os.path.join(ROOT, "tests", "root_all.cu"), "-o", out])
    return out


def test_root_program_builds(tmp_path):
    _build(tmp_path)


@pytest.mark.gpu
def test_root_of_every_number_is_rounded(tmp_path):
    r = subprocess.run([_build(tmp_path)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr
    assert r.stdout.split() == ["0", "0", "0"]
