"""Ranks of one process calling the operations on lists together: ranks that disagree
are refused before anything runs, and a host that runs out of memory leaves the group
usable."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

import adamw_ref as A

import coconet_b200 as coco

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
COUNTS = [1000, 7, 257]
HYPER = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-6, weight_decay=0.01)


class Ranks:
    def __init__(self, quant, counts=COUNTS):
        self.quant = quant
        self.comms = coco.Communicator.init_all(2, [0, 0])
        self.ws = [[torch.ones(c, device="cuda") for c in counts] for _ in range(2)]
        self.gs = [[torch.full((c,), 0.5, device="cuda") for c in counts] for _ in range(2)]
        if quant:
            self.state = [coco.quant_state(counts, 2) for _ in range(2)]
        else:
            n = coco.scattered_slice_elems(counts, 2)
            self.state = [tuple(torch.zeros(n, device="cuda") for _ in range(2)) for _ in range(2)]

    def step(self, *by_rank):
        with coco.group():
            for r, kw in enumerate(by_rank):
                kw = dict(HYPER, step=2, grad_scale=1.0, norm=None, no_decay=None, **({"seed": 5} if self.quant else {})) | kw
                call = self.comms[r].fused_adamw_quant_scattered if self.quant else self.comms[r].fused_adamw_scattered
                call(self.gs[r], self.ws[r], *self.state[r], **kw)

    def untouched(self):
        torch.cuda.synchronize()
        return (all(bool((x == 1).all()) for r in self.ws for x in r) and
                all(not x.view(torch.uint8).any() for r in self.state for x in r))


@pytest.fixture
def ranks(request):
    r = Ranks(getattr(request, "param", False))
    yield r
    torch.cuda.synchronize()
    for c in r.comms:
        c.destroy()


@pytest.mark.gpu
@pytest.mark.parametrize("ranks", [False, True], indirect=True, ids=["fp32", "8-bit"])
def test_ranks_that_disagree_about_a_step_are_refused(ranks):
    norm = torch.tensor([2.0, 0.5], device="cuda")
    cases = [dict(lr=2e-3), dict(beta1=0.8), dict(beta2=0.99), dict(eps=1e-5), dict(weight_decay=0.02), dict(step=3),
             dict(grad_scale=0.5), dict(norm=norm), dict(no_decay=[True, False, False])]
    if ranks.quant:
        cases += [dict(seed=6), dict(seed=5 + (1 << 32))]
    for kw in cases:
        for by_rank in (({}, kw), (kw, {})):
            with pytest.raises(coco.CocoError) as e:
                ranks.step(*by_rank)
            assert e.value.code == 2, kw
            assert ranks.untouched(), kw
    ranks.step(dict(norm=norm, no_decay=[False] * 3), dict(norm=norm.clone()))   # the same in other words
    assert not ranks.untouched()
    assert all(torch.equal(a, b) for a, b in zip(*ranks.ws))
    assert all(c.status()["code"] == 0 for c in ranks.comms)


@pytest.mark.gpu
def test_ranks_that_disagree_about_a_norm_are_refused(ranks):
    outs = [torch.full((2,), -1.0, device="cuda") for _ in range(2)]

    def norm(*by_rank):
        with coco.group():
            for r, kw in enumerate(by_rank):
                ranks.comms[r].grad_norm_scattered(ranks.gs[r], outs[r], **kw)
    for kw in (dict(max_norm=1.0), dict(grad_scale=0.5)):
        for by_rank in (({}, kw), (kw, {})):
            with pytest.raises(coco.CocoError) as e:
                norm(*by_rank)
            assert e.value.code == 2, kw
    torch.cuda.synchronize()
    assert all(bool((o == -1).all()) for o in outs)
    norm(dict(max_norm=1.0), dict(max_norm=1.0))
    n = float(np.sqrt(sum(COUNTS)))     # the sum of the two gradients is 1 everywhere
    for o in outs:
        assert abs(float(o[0]) - n) <= 1.1 * A.U * n and abs(float(o[1]) - 1 / n) <= 2.1 * A.U / n


@pytest.mark.gpu
@pytest.mark.parametrize("late", [0, 1])
@pytest.mark.parametrize("op", ["norm", "fp32", "8-bit"])
def test_ranks_of_one_gpu_with_a_stream_each(op, late):
    """The gradients of one rank come late on its stream, and its stream reads the results at once."""
    counts = [70001, 513, 9]
    ranks = Ranks(op == "8-bit", counts)
    try:
        streams = [torch.cuda.Stream() for _ in range(2)]
        outs = [torch.zeros(2, device="cuda") for _ in range(2)]
        a = torch.ones(4096, 4096, device="cuda")
        b = torch.empty_like(a)
        seen = [None, None]
        for value in (1.5, 3.5):
            torch.cuda.synchronize()
            with torch.cuda.stream(streams[late]):
                for _ in range(20):             # some milliseconds
                    torch.matmul(a, a, out=b)
                for g in ranks.gs[late]:
                    g.fill_(value)
            with coco.group():
                for r in range(2):
                    if op == "norm":
                        ranks.comms[r].grad_norm_scattered(ranks.gs[r], outs[r], stream=streams[r])
                    elif op == "fp32":
                        ranks.comms[r].fused_adamw_scattered(ranks.gs[r], ranks.ws[r], *ranks.state[r], **HYPER, step=0,
                                                             stream=streams[r])
                    else:
                        ranks.comms[r].fused_adamw_quant_scattered(ranks.gs[r], ranks.ws[r], *ranks.state[r], **HYPER,
                                                                   step=0, seed=1, stream=streams[r])
            for r in range(2):
                with torch.cuda.stream(streams[r]):
                    seen[r] = [x.clone() for x in (outs[r:r + 1] if op == "norm" else ranks.ws[r])]
                    for g in ranks.gs[r]:
                        g.fill_(0.5)            # the next step's, while the other rank may still be at it
            torch.cuda.synchronize()
            if op == "norm":
                n = (0.5 + value) * sum(counts) ** 0.5
                assert all(abs(float(s[0][0]) - n) <= 1.1 * A.U * n for s in seen)
            else:
                assert all(torch.equal(x, y) for r in range(2) for x, y in zip(seen[r], ranks.ws[r]))
                assert all(torch.equal(x, y) for x, y in zip(*ranks.ws))
        if op == "fp32":    # both steps saw the late gradients: m = 0.1 (0.9 * 2 + 4), where the fp32 number
            m = torch.cat([x for r in ranks.state for x in r[:1]])   # 1 - 0.9 is 4 u off, and four roundings more
            assert abs(float(m.max()) - 0.58) <= 8 * A.U * 0.58
        assert all(c.status()["code"] == 0 for c in ranks.comms)
    finally:
        torch.cuda.synchronize()
        for c in ranks.comms:
            c.destroy()


OUT_OF_MEMORY = f"""
import ctypes as C, sys
sys.path[:0] = [{os.path.dirname(os.path.abspath(__file__))!r}, {ROOT!r}]
import torch, coconet_b200 as coco
from test_list_group_gpu import Ranks
shim = C.CDLL(sys.argv[1])
shim.new_fails_at.argtypes = [C.c_size_t, C.c_int]
ranks = Ranks(sys.argv[2] == "8-bit", [100] * 41)
failed = 0
for skip in range(64):
    # the tables that a launch is made from hold 24 bytes for each of the 41 tensors
    shim.new_fails_at(24 * 41, skip)
    try:
        ranks.step({{}}, {{}})
        code = 0
    except coco.CocoError as e:
        code = e.code
    hit = shim.new_failed()
    shim.new_fails_at(0, 0)
    assert code == (7 if hit else 0), (skip, code, hit)
    if not hit:
        break
    failed += 1
    assert ranks.untouched(), skip
assert failed > 0
torch.cuda.synchronize()
assert not ranks.untouched()
ranks.step({{}}, {{}})                 # and once more, as ever
torch.cuda.synchronize()
assert all(c.status()["code"] == 0 for c in ranks.comms)
print("failed", failed)
"""


@pytest.mark.gpu
@pytest.mark.parametrize("form", ["fp32", "8-bit"])
def test_a_host_out_of_memory_leaves_the_group_usable(tmp_path, form):
    shim = str(tmp_path / "new_fails.so")
    subprocess.check_call(["g++", "-O1", "-fPIC", "-shared", os.path.join(ROOT, "tests", "new_fails.cpp"), "-o", shim])
    r = subprocess.run([sys.executable, "-c", OUT_OF_MEMORY, shim, form], env=dict(os.environ, LD_PRELOAD=shim),
                       capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-3000:]
