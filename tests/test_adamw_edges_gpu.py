"""AdamW over lists at the ends of its ranges: moments up to the largest fp32 number in
8 bits, steps of the 8-bit form in a row against the scalar evaluation, long lists of
large tensors."""
import numpy as np
import pytest
import torch

import adamw_ref as A
from test_adamw_gpu import H, RAGGED, TYPES, _aligned, _lp_of, _make, _norm64, comm  # noqa: F401

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


# ---- steps in a row -----------------------------------------------------------------------
@pytest.mark.parametrize("capture", [False, True])
def test_quant_steps_in_a_row_bit_for_bit(comm, capture):  # noqa: F811
    """Norm and 8-bit AdamW, clipped, three steps from the zero state, plain or as captured graphs: every step's codes
    and scales are those of the scalar evaluation that goes on from the step before, with the norm as it was returned."""
    counts = RAGGED
    off, total = A.starts(counts, 256)
    w, _, _, _ = _make(counts, 130, "bf16", step=0)
    ws, gs = _aligned(w, torch.float32), [torch.zeros(c, dtype=torch.bfloat16, device="cuda") for c in counts]
    lps = [x.bfloat16() for x in ws]
    no_decay = [c < 100 for c in counts]
    lst = coco.TensorList(gs, ws, lps=lps, no_decay=no_decay)
    st, norm = coco.quant_state(counts, 1), torch.zeros(2, device="cuda")
    state = [(np.zeros(c, np.uint8), np.zeros(c, np.uint8), np.zeros((-(-c // 256), 2), np.uint8)) for c in counts]

    def step(k):
        comm.grad_norm_scattered(lst, norm, max_norm=0.02, grad_scale=0.5)
        comm.fused_adamw_quant_scattered(lst, None, *st, H["lr"], H["beta1"], H["beta2"], H["eps"], H["weight_decay"], k, 15,
                                         grad_scale=0.5, norm=norm)
    for k in range(3):
        _, _, _, (g,) = _make(counts, 140 + k, "bf16")
        for t, x in zip(gs, g):
            t.copy_(torch.from_numpy(x))
        if capture:
            graph = torch.cuda.CUDAGraph()
            torch.cuda.synchronize()
            with torch.cuda.graph(graph):
                step(k)
            graph.replay()
        else:
            step(k)
        torch.cuda.synchronize()
        n, clip = norm.tolist()
        assert abs(n - _norm64(g, 0.5)) <= 5.1 * A.U * n and clip < 1   # it is clipped
        s = A.factor32(0.5, (n, clip))
        gm, gr, gsc = _state_bytes(st)
        for b, c in enumerate(counts):
            if c == 0:
                continue
            mc, rc, sc = state[b]
            scaled = g[b].astype(np.float32) * s
            old = (A.code_values(mc) * A.scale_values(sc[:, 0]).repeat(256)[:c],
                   (A.code_values(rc) * A.scale_values(sc[:, 1]).repeat(256)[:c]) ** 2)
            _, mc, rc, sc, _, _ = A.quant_step32(w[b], mc, rc, sc, scaled, k, 15, off[b], not no_decay[b])
            state[b] = (mc, rc, sc)
            assert np.array_equal(gm[off[b]:off[b] + c], mc), (k, b)
            assert np.array_equal(gr[off[b]:off[b] + c], rc), (k, b)
            assert np.array_equal(gsc[off[b] // 256:off[b] // 256 + len(sc)], sc), (k, b)
            before, now = w[b].astype(np.float64), ws[b].cpu().numpy()
            x = (before, old[0], old[1], scaled.astype(np.float64), k, not no_decay[b])
            new, _, _, q = A.step64(*x)
            assert (np.abs(now - new) <= A.bounds64(*x)[0]).all(), (k, b)
            assert (np.abs(now - before)[np.abs(q) > 1e-5] > 0).all(), (k, b)   # the weights did move
            w[b] = now
            assert np.array_equal(lps[b].float().cpu().numpy(), _lp_of(now, "bf16")), (k, b)


# ---- long lists of large tensors ------------------------------------------------------------
def _encode_on_gpu(x, bits16):
    """adamw_ref.encode32 for whole blocks [n, 256], with torch."""
    e = (x.abs().amax(1).view(torch.int32) >> 23).clamp(8, 254)
    y = (x.abs() * ((261 - e) << 23).view(torch.float32)[:, None]) * 2.0 ** -120
    code = (y.view(torch.int32) + ((bits16 << 4) | 8)) >> 20
    return code | ((x.view(torch.int32) >> 24) & 0x80), e - 7


@pytest.mark.parametrize("gt,lp", [("bf16", "bf16"), ("f32", None)])
def test_quant_adamw_of_a_long_list_of_large_tensors(comm, gt, lp):  # noqa: F811
    """A list like a model's: more than 64 tensors, 1024 and more units each on average.  Codes and scales bit for bit,
    weights within the bound of their roundings."""
    counts = [262144 + 256 * (k % 3) for k in range(70)] + [300, 1, 255, 4194304]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert len(counts) > 64 and sum(-(-c // 256) for c in counts) >= max(1024 * len(counts), 8 * 24 * sms)
    off, total = A.starts(counts, 256)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(7)
    g, w = (torch.zeros(total, device="cuda") for _ in range(2))
    live = torch.zeros(total, dtype=torch.bool, device="cuda")
    for o, c in zip(off, counts):
        live[o:o + c] = True
    g[live] = (torch.randn(int(live.sum()), device="cuda", generator=gen) * 1e-3).to(TYPES[gt]).float()
    w[live] = torch.randn(int(live.sum()), device="cuda", generator=gen) * 0.02
    gs = [g[o:o + c].to(TYPES[gt]) for o, c in zip(off, counts)]
    ws = [w[o:o + c].clone() for o, c in zip(off, counts)]
    lps = [torch.zeros(c, dtype=TYPES[lp], device="cuda") for c in counts] if lp else None
    st = coco.quant_state(counts, 1)
    key = 33
    m, r = torch.zeros(total, device="cuda"), torch.zeros(total, device="cuda")
    for step in (0, 1):
        comm.fused_adamw_quant_scattered(gs, ws, *st, H["lr"], H["beta1"], H["beta2"], H["eps"], H["weight_decay"], step, key, w_lps=lps)
        h = {k: float(x) for k, x in A.scalars32(step, **A.HYPER).items()}
        m = m * h["b1"] + g * h["omb1"]
        r = torch.sqrt((r * r) * h["b2"] + (g * g) * h["omb2"])
        q = ((m.double() * h["c1"]) / (r.double() * h["rs2"] + h["eps"]))
        new = w.double() * h["decay"] - q
        bits = torch.from_numpy(A.rounding_bits(0, total, key, step).astype(np.int64)).cuda()
        mc, ms = _encode_on_gpu(m.view(-1, 256), (bits & 0xFFFF).to(torch.int32).view(-1, 256))
        rc, rs = _encode_on_gpu(r.view(-1, 256), (bits >> 16).to(torch.int32).view(-1, 256))
        rc = torch.where(r.view(-1, 256) > 0, rc.clamp_min(1), rc)
        mc, rc = (x.view(-1).to(torch.uint8) for x in (mc, rc))
        for want, got in ((mc, st[0]), (rc, st[1])):
            assert torch.equal(torch.where(live, want, 0), got.view(torch.uint8)), step
        assert torch.equal(torch.stack([ms, rs], 1).to(torch.uint8), st[2].view(torch.uint8)), step
        got = torch.zeros_like(w)
        for o, c, x in zip(off, counts, ws):
            got[o:o + c] = x
        # near32's count: 8 u of the update, and the last difference half a step on either side
        assert bool(((got.double() - new).abs() <= 8 * A.U * q.abs() + 2 * A.U * new.abs() + 2.0 ** -140)[live].all()), step
        if lp:
            assert all(torch.equal(x, y.to(TYPES[lp])) for x, y in zip(lps, ws)), step
        w = got
        m, r = (coco.quant_decode(*st)[0], coco.quant_decode(*st)[1].sqrt())
