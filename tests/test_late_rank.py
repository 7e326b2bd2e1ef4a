"""A rank whose CTAs disagree on whether a peer came in time (tests/late_rank.cu): the
part of a gradient norm that is missing must not pass for a norm, and a step that is
missing a part must not be announced as complete.  CPU: the program compiles for
sm_100a against the library.  GPU: every wait in it is bounded."""
import json
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NVCC = os.environ.get("NVCC", "/usr/local/cuda/bin/nvcc")
LIBDIR = os.path.join(ROOT, "coconet_b200")


def _build(out):
    assert os.path.exists(os.path.join(LIBDIR, "libcoconet_rt.so")), "build the library first"
    subprocess.check_call([NVCC, "-gencode", "arch=compute_100a,code=sm_100a", "-O2", "-std=c++17",
                           "-I", os.path.join(ROOT, "include"), "-I", os.path.join(LIBDIR, "csrc"),
                           os.path.join(ROOT, "tests", "late_rank.cu"), "-o", out,
                           "-L", LIBDIR, "-lcoconet_rt", "-Xlinker", "-rpath", "-Xlinker", LIBDIR])
    return out


def test_late_rank_program_builds(tmp_path):
    _build(str(tmp_path / "late_rank"))


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    return _build(str(tmp_path_factory.mktemp("late") / "late_rank"))


def _run(program, *args):
    r = subprocess.run([program, *args], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stdout + r.stderr
    out = json.loads(r.stdout)
    assert out["counters"] == 0   # left ready for the next call
    return {k: float.fromhex(x) if isinstance(x, str) else x for k, x in out.items()}


@pytest.mark.gpu
def test_norm_with_a_rank_in_time(program):
    out = _run(program, "norm", "in-time")
    n = 2.0 * out["n"] ** 0.5      # the sum over two ranks is 2 everywhere; exact in fp64
    assert out["status"] == 0 and abs(out["norm"] - n) <= 2.0 ** -24 * n
    assert out["told_norm"] == 1 and out["told_part"] == 4.0 * out["n"]


@pytest.mark.gpu
def test_norm_that_lost_a_part_is_no_number(program):
    out = _run(program, "norm")
    assert out["status"] == 5 and out["phase"] == 1
    assert out["norm"] != out["norm"] and out["clip"] == 0.0, out   # nan: the step that reads it is skipped
    if out["told_norm"]:           # what the peer adds up is no number either
        assert out["told_part"] != out["told_part"], out


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["adamw", "adamw8"])
def test_step_with_a_rank_in_time(program, op):
    out = _run(program, op, "in-time")
    assert out["status"] == 0 and out["stepped"] == out["n"] and out["told_done"] == 1


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["adamw", "adamw8"])
def test_step_that_lost_a_part_is_not_announced_as_done(program, op):
    out = _run(program, op)
    assert out["status"] == 5 and out["phase"] == 1
    assert 0 < out["stepped"] < out["n"], out   # some CTAs gave up, others did not
    assert out["told_done"] == 0, out           # the peer's wait runs out: its status says so too
