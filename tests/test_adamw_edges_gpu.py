"""AdamW over lists at the ends of its ranges: moments up to the largest fp32 number in
8 bits."""
import numpy as np
import pytest
import torch

import adamw_ref as A
from test_adamw_gpu import H, comm  # noqa: F401

pytestmark = pytest.mark.gpu

import coconet_b200 as coco  # noqa: E402


def _state_bytes(st):
    return [x.view(torch.uint8).cpu().numpy() for x in st]


# ---- blocks of large moments ----------------------------------------------------------
@pytest.mark.parametrize("top", [13, 14, 15, 60, 112, 113, 114, 115, 120, 126, 127])
@pytest.mark.parametrize("spread", [0, 20, 200])
def test_quant_codes_of_large_first_moments(comm, top, spread):  # noqa: F811
    """beta1 = 0: m is the gradient, up to just below 2^(top + 1); codes and scales bit for bit."""
    n = 512
    r = np.random.default_rng(top * 1000 + spread)
    g = np.exp2(np.maximum(top - r.uniform(0, spread, n), -149.0)) * r.uniform(1, 1.99999, n) * r.choice([-1, 1], n)
    g[::97] = 1.99999 * 2.0 ** top
    g = np.clip(g, -float(np.finfo(np.float32).max), float(np.finfo(np.float32).max)).astype(np.float32)
    hyper = dict(A.HYPER, beta1=A.F(0.0), weight_decay=A.F(0.0))
    w = torch.zeros(n, device="cuda")
    st = coco.quant_state([n], 1)
    comm.fused_adamw_quant_scattered([torch.from_numpy(g).cuda()], [w], *st, H["lr"], 0.0, H["beta2"], H["eps"], 0.0, 4, 21)
    zero = np.zeros(n, np.uint8)
    _, mc, rc, sc, m, _ = A.quant_step32(np.zeros(n, np.float32), zero, zero, np.zeros((2, 2), np.uint8), g, 4, 21, 0, hyper=hyper)
    got = _state_bytes(st)
    assert np.array_equal(m, g) and (sc[:, 0] != 255).all()
    assert np.array_equal(got[2], sc) and np.array_equal(got[1], rc)
    assert np.array_equal(got[0], mc), np.flatnonzero(got[0] != mc)[:8]


@pytest.mark.parametrize("scale", [234, 240, 246, 247])
def test_quant_codes_of_a_state_with_a_large_first_moment(comm, scale):  # noqa: F811
    """A finite state whose m is large beside an ordinary v: every moment stays finite, codes bit for bit."""
    n = 700
    r = np.random.default_rng(scale)
    mc = r.integers(0, 0x70, n).astype(np.uint8) | (r.integers(0, 2, n) * 0x80).astype(np.uint8)
    rc = r.integers(1, 0x78, n).astype(np.uint8)
    sc = np.stack([np.full(3, scale), np.full(3, 110)], 1).astype(np.uint8)
    g = r.normal(0, 1e-3, n).astype(np.float32)
    st = coco.quant_state([n], 1)
    for x, y in zip(st, (mc, rc, sc)):
        flat = x.view(torch.uint8).view(-1)
        flat[:y.size] = torch.from_numpy(y.reshape(-1)).cuda()
    w = torch.zeros(n, device="cuda")
    for step in (10, 11):
        comm.fused_adamw_quant_scattered([torch.from_numpy(g).cuda()], [w], *st, 0.0, H["beta1"], H["beta2"], H["eps"], 0.0, step, 5)
        hyper = dict(A.HYPER, lr=A.F(0.0), weight_decay=A.F(0.0))
        _, mc, rc, sc, m, v = A.quant_step32(np.zeros(n, np.float32), mc, rc, sc, g, step, 5, 0, hyper=hyper)
        got = _state_bytes(st)
        assert np.isfinite(m).all() and np.isfinite(v).all() and (sc != 255).all()
        assert np.array_equal(got[2], sc) and np.array_equal(got[1][:n], rc)
        assert np.array_equal(got[0][:n], mc), (step, np.flatnonzero(got[0][:n] != mc)[:8])


@pytest.mark.parametrize("top", [13, 14, 40, 62, 63])
def test_quant_codes_of_large_roots(comm, top):  # noqa: F811
    """beta2 = 0: the root is the gradient's magnitude, up to the root of the largest number; none is stored as 0."""
    n = 512
    r = np.random.default_rng(top)
    g = (np.exp2(np.maximum(top - r.uniform(0, 80, n), -60.0)) * r.uniform(1, 1.999, n)).astype(np.float32)
    g[::51] = np.float32(1.999 * 2.0 ** top)
    w = torch.zeros(n, device="cuda")
    st = coco.quant_state([n], 1)
    comm.fused_adamw_quant_scattered([torch.from_numpy(g).cuda()], [w], *st, H["lr"], H["beta1"], 0.0, H["eps"], 0.0, 4, 22)
    zero = np.zeros(n, np.uint8)
    hyper = dict(A.HYPER, beta2=A.F(0.0), weight_decay=A.F(0.0))
    _, mc, rc, sc, _, _ = A.quant_step32(np.zeros(n, np.float32), zero, zero, np.zeros((2, 2), np.uint8), g, 4, 22, 0, hyper=hyper)
    got = _state_bytes(st)
    assert np.array_equal(got[2], sc) and np.array_equal(got[0], mc) and np.array_equal(got[1], rc)
    assert (got[1] > 0).all() and (sc != 255).all()
