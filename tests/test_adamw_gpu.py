"""AdamW over lists of tensors (fp32 and 8-bit moments) and the gradient norm, on
the GPU: against evaluations in fp64 with bounds counted from the roundings, bit
for bit against fp32 evaluations, one rank and virtual ranks."""
import math

import numpy as np
import pytest
import torch

import adamw_ref as A

pytestmark = pytest.mark.gpu

import coconet_b200 as coco  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
H = {k: float(v) for k, v in A.HYPER.items()}
# sizes around groups of 8, blocks of 256 and a warp's unit; tensors that share a unit; empty ones
RAGGED = [1000, 8, 3, 0, 4096, 70001, 2, 1, 255, 256, 257, 24, 0, 7, 9, 511, 513, 31, 33]
LISTS = {
    "one element": [1],
    "seven": [7],
    "one unit": [256],
    "ragged": RAGGED,
    "many small": [1 + (k * 37) % 61 for k in range(1100)],   # more than one launch holds
    "long and short": [300001] + [5] * 70 + [65536],
}


@pytest.fixture
def comm():
    c = coco.Communicator.init_all(1, [0])[0]
    yield c
    torch.cuda.synchronize()
    assert c.status()["code"] == 0
    c.destroy()


def _views(arrays, dtype, offset, gap, fill=7.0):
    """The arrays as views into one buffer: `offset` elements in front, `gap` between
    them; (buffer, views).  What lies between holds `fill`."""
    total = offset + sum(a.size + gap for a in arrays)
    buf = torch.full((total,), fill, dtype=dtype, device="cuda")
    at, out = offset, []
    for a in arrays:
        buf[at:at + a.size] = torch.from_numpy(a).to(dtype=dtype, device="cuda")
        out.append(buf[at:at + a.size])
        at += a.size + gap
    return buf, out


def _gaps_untouched(buf, views, fill=7.0):
    mask = torch.ones(buf.numel(), dtype=torch.bool, device="cuda")
    for v in views:
        at = (v.data_ptr() - buf.data_ptr()) // buf.element_size()
        mask[at:at + v.numel()] = False
    return bool((buf[mask] == fill).all())


def _aligned(arrays, dtype):
    return [torch.from_numpy(a).to(dtype=dtype, device="cuda") for a in arrays]


def _make(counts, seed, gt, ranks=1, step=3):
    """Weights, moments and per-rank gradients (exact in gt), as fp32 arrays."""
    r = np.random.default_rng(seed)
    w = [r.normal(0, 0.02, c).astype(np.float32) for c in counts]
    zero = step == 0
    m = [np.zeros(c, np.float32) if zero else r.normal(0, 3e-4, c).astype(np.float32) for c in counts]
    v = [np.zeros(c, np.float32) if zero else (np.exp(r.normal(0, 1, c)) * 1e-6).astype(np.float32) for c in counts]
    g = []
    for _ in range(ranks):
        one = []
        for c in counts:
            x = r.normal(0, 1e-3, c) * (r.random(c) > 0.1)
            one.append(torch.from_numpy(x).to(TYPES[gt]).float().numpy())
        g.append(one)
    return w, m, v, g


def _flat(parts, counts, align, slack=0, fill=0.0):
    off, total = A.starts(counts, align)
    x = np.full(total + slack, fill, parts[0].dtype if parts else np.float32)
    for o, p in zip(off, parts):
        x[o:o + p.size] = p
    return x


def _lp_of(w, lp):
    return torch.from_numpy(w).to(TYPES[lp]).float().numpy()


@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("gt,lp", [("f32", None), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("bf16", None)])
@pytest.mark.parametrize("layout", ["aligned", "packed", "gaps"])
def test_adamw_against_fp64(comm, name, gt, lp, layout):
    counts, step, scale = LISTS[name], 3, 0.5
    w, m, v, (g,) = _make(counts, 1, gt, step=step)
    no_decay = [k % 3 == 1 for k in range(len(counts))]
    gs, ws = (_aligned(g, TYPES[gt]), _aligned(w, torch.float32)) if layout == "aligned" else (None, None)
    off, gap = {"packed": (0, 0), "gaps": (1, 3)}.get(layout, (0, 0))
    bufs = []
    lps = None
    if layout != "aligned":
        gb, gs = _views(g, TYPES[gt], off, gap)
        wb, ws = _views(w, torch.float32, off, gap)
        bufs = [(gb, gs), (wb, ws)]
    if lp:
        if layout == "aligned":
            lps = [torch.zeros(c, dtype=TYPES[lp], device="cuda") for c in counts]
        else:
            lb, lps = _views([np.zeros(c, np.float32) for c in counts], TYPES[lp], off, gap)
            bufs.append((lb, lps))
    # one element past an aligned start: the state itself may be unaligned too
    shift = 1 if layout == "gaps" else 0
    ma = torch.from_numpy(np.concatenate([np.zeros(shift, np.float32), _flat(m, counts, 8, slack=16, fill=5.0)])).cuda()[shift:]
    va = torch.from_numpy(np.concatenate([np.zeros(shift, np.float32), _flat(v, counts, 8, slack=16, fill=5.0)])).cuda()[shift:]
    comm.fused_adamw_scattered(gs, ws, ma, va, H["lr"], H["beta1"], H["beta2"], H["eps"], H["weight_decay"], step,
                               w_lps=lps, no_decay=no_decay, grad_scale=scale)
    torch.cuda.synchronize()
    places, total = A.starts(counts, 8)
    ma, va = ma.cpu().numpy(), va.cpu().numpy()
    assert (ma[total:] == 5.0).all() and (va[total:] == 5.0).all()
    for b, c in enumerate(counts):
        dec = not no_decay[b]
        args = (w[b].astype(np.float64), m[b].astype(np.float64), v[b].astype(np.float64), g[b].astype(np.float64) * scale)
        rw, rm, rv, _ = A.step64(*args, step, dec)
        ew, em, ev = A.bounds64(*args, step, dec)
        got = ws[b].cpu().numpy()
        assert (np.abs(got - rw) <= ew).all(), (b, np.abs(got - rw).max())
        assert (np.abs(ma[places[b]:places[b] + c] - rm) <= em).all(), b
        assert (np.abs(va[places[b]:places[b] + c] - rv) <= ev).all(), b
        if lp:   # the copy is the weight rounded once
            assert np.array_equal(lps[b].float().cpu().numpy(), _lp_of(got, lp)), b
    for buf, views in bufs:
        assert _gaps_untouched(buf, views)


@pytest.mark.parametrize("R", [1, 2, 3, 8])
@pytest.mark.parametrize("gt,lp", [("f32", None), ("f16", "f16"), ("bf16", "bf16")])
@pytest.mark.parametrize("packed", [False, True])
def test_adamw_bit_for_bit_on_every_rank_count(R, gt, lp, packed):
    counts = RAGGED if R > 1 else LISTS["long and short"]
    comms = coco.Communicator.init_all(R, [0] * R)
    S = coco.scattered_slice_elems(counts, R)
    assert S == A.slice_elems(counts, R, 8)
    off, total = A.starts(counts, 8)
    try:
        w, m, v, _ = _make(counts, 2, gt, step=1)
        fm, fv = _flat(m, counts, 8), _flat(v, counts, 8)
        pad = np.zeros(R * S - total, np.float32)
        ms = [torch.from_numpy(x).cuda() for x in np.split(np.concatenate([fm, pad]), R)]
        vs = [torch.from_numpy(x).cuda() for x in np.split(np.concatenate([fv, pad]), R)]
        make = (lambda a, t: _views(a, t, 1, 0)[1]) if packed else _aligned
        ws = [make(w, torch.float32) for _ in range(R)]
        lps = [make([np.zeros(c, np.float32) for c in counts], TYPES[lp]) if lp else None for _ in range(R)]
        for step in (1, 2):
            _, _, _, g = _make(counts, 10 + step, gt, ranks=R)
            norm = torch.tensor([2.0, 0.75], device="cuda")
            gs = [make(g[r], TYPES[gt]) for r in range(R)]
            with coco.group():
                for r, c in enumerate(comms):
                    c.fused_adamw_scattered(gs[r], ws[r], ms[r], vs[r], H["lr"], H["beta1"], H["beta2"], H["eps"],
                                            H["weight_decay"], step, w_lps=lps[r], grad_scale=0.25, norm=norm)
            torch.cuda.synchronize()
            s = A.factor32(0.25, (2.0, 0.75))
            for c in comms:
                assert c.status()["code"] == 0
            gm = np.concatenate([x.cpu().numpy() for x in ms])
            gv = np.concatenate([x.cpu().numpy() for x in vs])
            for b, c in enumerate(counts):
                gsum = A.sum32([g[r][b] for r in range(R)]) * s
                old = (w[b], m[b], v[b], gsum)
                _, m[b], v[b] = A.step32(*old, step)
                # the weights: the same on every rank (and, below, whatever the layout), near the fp32 evaluation
                lo = max(0, -off[b])
                w[b] = np.concatenate([ws[r][b].cpu().numpy()[max(0, r * S - off[b]):max(0, (r + 1) * S - off[b])]
                                       for r in range(R)])[lo:c] if lp else ws[0][b].cpu().numpy()
                assert w[b].size == c and A.near32(w[b], *old, step), (step, b)
                assert np.array_equal(gm[off[b]:off[b] + c], m[b]), (step, b)
                assert np.array_equal(gv[off[b]:off[b] + c], v[b]), (step, b)
                for r in range(R):
                    got = ws[r][b].cpu().numpy()
                    if lp:   # only the own slice of the fp32 weights is updated; the copy is everywhere
                        lo, hi = max(off[b], r * S) - off[b], min(off[b] + c, (r + 1) * S) - off[b]
                        assert lo >= hi or np.array_equal(got[lo:hi], w[b][lo:hi]), (step, b, r)
                        assert np.array_equal(lps[r][b].float().cpu().numpy(), _lp_of(w[b], lp)), (step, b, r)
                    else:
                        assert np.array_equal(got, w[b]), (step, b, r)
    finally:
        for c in comms:
            c.destroy()


def _quant_initial(counts, m, v, seed):
    """8-bit state of the given moments, tensor by tensor."""
    r = np.random.default_rng(seed)
    out = []
    for a, b in zip(m, v):
        mc, ms = A.encode32(a, r.integers(0, 1 << 16, a.size).astype(np.uint32))
        rc, rs = A.encode32(np.sqrt(b), r.integers(0, 1 << 16, b.size).astype(np.uint32))
        out.append((mc, rc, np.stack([ms, rs], 1)))
    return out


@pytest.mark.parametrize("quant", [False, True])
def test_layout_and_alignment_do_not_change_a_bit(comm, quant):
    """Vector, scalar and several-tensors-a-unit paths give the same bits."""
    counts = [70001, 4096, 255, 8, 1, 1000]
    w, m, v, (g,) = _make(counts, 9, "bf16")
    results = []
    for off, gap in ((0, 7), (1, 0), (3, 2)):
        ws = _views(w, torch.float32, off, gap)[1] if off else _aligned(w, torch.float32)
        gs = _views(g, torch.bfloat16, off, gap)[1] if off else _aligned(g, torch.bfloat16)
        if quant:
            st = coco.quant_state(counts, 1)
            for step in range(2):
                comm.fused_adamw_quant_scattered(gs, ws, *st, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.1, step, 11)
        else:
            st = [torch.from_numpy(_flat(x, counts, 8)).cuda() for x in (m, v)]
            comm.fused_adamw_scattered(gs, ws, *st, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.1, 3)
        results.append(ws + [x.view(torch.uint8) if quant else x for x in st])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


@pytest.mark.parametrize("R,name", [(1, n) for n in LISTS] + [(2, "ragged"), (3, "ragged"), (8, "ragged"), (2, "one element")])
@pytest.mark.parametrize("gt,lp,layout", [("f32", None, "aligned"), ("bf16", "bf16", "aligned"), ("f16", "f16", "packed"),
                                          ("bf16", None, "packed")])
def test_quant_adamw_bit_for_bit(R, name, gt, lp, layout):
    counts = LISTS[name]
    comms = coco.Communicator.init_all(R, [0] * R)
    S = coco.quant_slice_elems(counts, R)
    assert S == A.slice_elems(counts, R, 256)
    off, total = A.starts(counts, 256)
    seed = 0x123456789AB
    try:
        w, m, v, _ = _make(counts, 3, gt)
        state = _quant_initial(counts, m, v, 4)
        shift = 1 if layout == "packed" else 0   # codes need no alignment
        flat = np.full((2, R * S), 0x55, np.uint8)      # bytes of no element keep what they hold
        scales = np.full((R * S // 256, 2), 0x44, np.uint8)
        for b, (mc, rc, sc) in enumerate(state):
            flat[0, off[b]:off[b] + counts[b]], flat[1, off[b]:off[b] + counts[b]] = mc, rc
            scales[off[b] // 256:off[b] // 256 + len(sc)] = sc

        def up(x):
            return torch.from_numpy(np.concatenate([np.zeros(shift, np.uint8), x])).cuda()[shift:]
        ms, rs = [up(x) for x in np.split(flat[0], R)], [up(x) for x in np.split(flat[1], R)]
        scs = [torch.from_numpy(x.copy()).cuda() for x in np.split(scales, R)]
        make = (lambda a, t: _views(a, t, 1, 0)[1]) if layout == "packed" else _aligned
        ws = [make(w, torch.float32) for _ in range(R)]
        lps = [make([np.zeros(c, np.float32) for c in counts], TYPES[lp]) if lp else None for _ in range(R)]
        no_decay = [k % 2 == 0 for k in range(len(counts))]
        for step in (5, 6):
            _, _, _, g = _make(counts, 20 + step, gt, ranks=R)
            gs = [make(g[r], TYPES[gt]) for r in range(R)]
            with coco.group():
                for r, c in enumerate(comms):
                    c.fused_adamw_quant_scattered(gs[r], ws[r], ms[r], rs[r], scs[r], H["lr"], H["beta1"], H["beta2"],
                                                  H["eps"], H["weight_decay"], step, seed, w_lps=lps[r],
                                                  no_decay=no_decay, grad_scale=0.5)
            torch.cuda.synchronize()
            for c in comms:
                assert c.status()["code"] == 0
            gm, gr = (np.concatenate([x.cpu().numpy() for x in y]) for y in (ms, rs))
            gsc = np.concatenate([x.cpu().numpy() for x in scs])
            exact_w = [x.copy() for x in w]
            for b, c in enumerate(counts):
                if c == 0:
                    continue
                mc, rc, sc = state[b]
                gsum = A.sum32([g[r][b] for r in range(R)]) * np.float32(0.5)
                old = (A.code_values(mc) * A.scale_values(sc[:, 0]).repeat(256)[:c],
                       (A.code_values(rc) * A.scale_values(sc[:, 1]).repeat(256)[:c]) ** 2)
                before = exact_w[b].astype(np.float64)
                _, mc, rc, sc, mf, rf = A.quant_step32(w[b], mc, rc, sc, gsum, step, seed, off[b], not no_decay[b])
                state[b] = (mc, rc, sc)
                w[b] = np.concatenate([ws[r][b].cpu().numpy()[max(0, r * S - off[b]):max(0, (r + 1) * S - off[b])]
                                       for r in range(R)])[:c] if lp else ws[0][b].cpu().numpy()
                assert np.array_equal(gm[off[b]:off[b] + c], mc), (step, b)
                assert np.array_equal(gr[off[b]:off[b] + c], rc), (step, b)
                assert np.array_equal(gsc[off[b] // 256:off[b] // 256 + len(sc)], sc), (step, b)
                # and in fp64: the weights within the roundings' bound, the codes within one code step
                rw, rm, rv, _ = A.step64(before, old[0], old[1], gsum.astype(np.float64), step, not no_decay[b])
                ew, _, _ = A.bounds64(before, old[0], old[1], gsum.astype(np.float64), step, not no_decay[b])
                assert (np.abs(w[b] - rw) <= ew).all(), (step, b)
                for codes, scale, x in ((mc, sc[:, 0], rm), (rc, sc[:, 1], np.sqrt(rv))):
                    s = A.scale_values(scale).repeat(256)[:c]
                    y = np.abs(x) / s
                    code_step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(y, 2.0 ** -6))), -6) - 3)
                    assert (np.abs(A.code_values(codes) * s - x) <= 1.001 * code_step * s).all(), (step, b)
                for r in range(R):
                    got = ws[r][b].cpu().numpy()
                    lo, hi = max(off[b], r * S) - off[b], min(off[b] + c, (r + 1) * S) - off[b]
                    if lp:
                        assert lo >= hi or np.array_equal(got[lo:hi], w[b][lo:hi]), (step, b, r)
                        assert np.array_equal(lps[r][b].float().cpu().numpy(), _lp_of(w[b], lp)), (step, b, r)
                    else:
                        assert np.array_equal(got, w[b]), (step, b, r)
            used = np.zeros(R * S, bool)
            for o, c in zip(off, counts):
                used[o:o + c] = True
            assert (gm[~used] == 0x55).all() and (gr[~used] == 0x55).all()
            assert (gsc[~used.reshape(-1, 256).any(1)] == 0x44).all()
    finally:
        for c in comms:
            c.destroy()


def test_quant_rounding_is_right_on_average(comm):
    """512 seeds round the same moments: every mean lies within 5 standard errors of the value (a rounding's
    deviation is at most half a code step), and the zero state decodes to zeros."""
    n, seeds = 1024, 512
    w0 = torch.zeros(n, device="cuda")
    g = torch.linspace(-1e-3, 2e-3, n, device="cuda")
    m_sum, r_sum = np.zeros(n), np.zeros(n)
    m0, r0, s0 = coco.quant_state([n], 1)
    assert float(coco.quant_decode(m0, r0, s0)[0].abs().sum()) == 0.0
    for seed in range(seeds):
        m, r, s = coco.quant_state([n], 1)
        comm.fused_adamw_quant_scattered([g], [w0.clone()], m, r, s, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.0, 0, seed)
        a, b = coco.quant_decode(m, r, s)
        m_sum += a.double().cpu().numpy()
        r_sum += b.double().sqrt().cpu().numpy()
    h = A.scalars32(0, **A.HYPER)
    gm = g.cpu().numpy()
    with np.errstate(all="ignore"):
        x, v = A.moments32(h, np.zeros(n, np.float32), np.zeros(n, np.float32), gm)
    for mean, val, floor in ((m_sum / seeds, x.astype(np.float64), 0.0), (r_sum / seeds, np.sqrt(v.astype(np.float64)), 2.0 ** -9)):
        scale = np.exp2(np.floor(np.log2(np.abs(val).reshape(-1, 256).max(1))) - 7).repeat(256)
        # a positive root below the smallest code, 2^-9, is that code whichever way it is rounded: 0 is raised to it
        val = np.where(val != 0, np.sign(val) * np.maximum(np.abs(val), floor * scale), 0.0)
        y = np.maximum(np.abs(val) / scale, 2.0 ** -6)
        code_step = np.exp2(np.floor(np.log2(y)) - 3) * scale
        assert (np.abs(mean - val) <= 5 * code_step / 2 / math.sqrt(seeds) + code_step * 2.0 ** -16).all()


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("bad", [math.inf, math.nan, -math.inf])
def test_a_norm_that_is_not_finite_skips_the_step(comm, quant, bad):
    counts = RAGGED
    w, m, v, (g,) = _make(counts, 5, "f32")
    ws, gs = _aligned(w, torch.float32), _aligned(g, torch.float32)
    lps = [torch.full((c,), 3.0, dtype=torch.bfloat16, device="cuda") for c in counts]
    norm = torch.tensor([bad, 0.0], device="cuda")
    if quant:
        st = [torch.randint(0, 0x78, (coco.quant_slice_elems(counts, 1),), dtype=torch.uint8, device="cuda") for _ in range(2)]
        st.append(torch.full((st[0].numel() // 256, 2), 100, dtype=torch.uint8, device="cuda"))
        before = [x.clone() for x in st]
        comm.fused_adamw_quant_scattered(gs, ws, *st, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.1, 3, 9, w_lps=lps, norm=norm)
    else:
        st = [torch.from_numpy(_flat(x, counts, 8)).cuda() for x in (m, v)]
        before = [x.clone() for x in st]
        comm.fused_adamw_scattered(gs, ws, *st, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.1, 3, w_lps=lps, norm=norm)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(st, before))
    assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(ws, w))
    assert all(bool((x == 3.0).all()) for x in lps)


def test_inf_and_nan_gradients_stay_where_they_are(comm):
    """Without a norm: fp32 moments carry inf and nan element by element, 8-bit ones mark the block."""
    n = 1024
    g = torch.full((n,), 1e-3, device="cuda")
    g[3], g[300], g[301] = math.nan, math.inf, -math.inf
    w, m, v = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    comm.fused_adamw_scattered([g], [w], m, v, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.0, 0)
    ok = torch.ones(n, dtype=torch.bool, device="cuda")
    ok[[3, 300, 301]] = False
    assert torch.isfinite(w[ok]).all() and not torch.isfinite(w[~ok]).any()
    assert torch.isfinite(m[ok]).all() and torch.isnan(m[3]) and m[300] == math.inf and m[301] == -math.inf
    w8 = torch.zeros(n, device="cuda")
    st = coco.quant_state([n], 1)
    comm.fused_adamw_quant_scattered([g], [w8], *st, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.0, 0, 1)
    a, b = coco.quant_decode(*st)
    assert torch.equal(w8[ok], w[ok]) and not torch.isfinite(w8[~ok]).any()
    assert torch.isnan(a[:512]).all() and torch.isnan(b[:512]).all()
    assert torch.isfinite(a[512:]).all() and torch.isfinite(b[512:]).all() and (b[512:] > 0).all()


def test_quant_extremes_of_a_block(comm):
    """Gradients from the smallest to the largest fp32 numbers in one block, bit for bit; a positive root of
    the second moment stays positive."""
    n = 512
    r = np.random.default_rng(8)
    g = (np.exp2(r.uniform(-149, 60, n)) * r.choice([-1, 1], n)).astype(np.float32)
    g[256:] = np.exp2(r.uniform(-149, -130, 256)).astype(np.float32)   # a block of subnormal numbers only
    w = torch.zeros(n, device="cuda")
    st = coco.quant_state([n], 1)
    ref = (np.zeros(n, np.float32), np.zeros(n, np.uint8), np.zeros(n, np.uint8), np.zeros((2, 2), np.uint8))
    for step in range(3):
        comm.fused_adamw_quant_scattered([torch.from_numpy(g).cuda()], [w], *st, H["lr"], H["beta1"], H["beta2"], H["eps"],
                                         0.0, step, 77)
        out = A.quant_step32(*ref, g, step, 77, 0, hyper=dict(A.HYPER, weight_decay=0.0))
        w_old, ref = ref[0], out[:4]
        assert np.array_equal(st[0].view(torch.uint8).cpu().numpy(), ref[1]), step
        assert np.array_equal(st[1].view(torch.uint8).cpu().numpy(), ref[2]), step
        assert np.array_equal(st[2].view(torch.uint8).cpu().numpy(), ref[3]), step
        got = w.cpu().numpy()
        q = np.abs(ref[0].astype(np.float64) - w_old)   # near32's bound; the update is what w lost
        assert (np.abs(got - ref[0].astype(np.float64)) <= 8 * A.U * (q + np.abs(ref[0])) + 2.0 ** -140).all(), step
        ref = (got,) + ref[1:]
        assert (ref[2][out[5] > 0] > 0).all()


# ---- the norm --------------------------------------------------------------------
def _norm64(gs, scale=1.0):
    return math.sqrt(math.fsum(float(x) ** 2 for g in gs for x in g.astype(np.float64))) * abs(scale)


@pytest.mark.parametrize("name", list(LISTS))
@pytest.mark.parametrize("gt", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["aligned", "packed", "gaps"])
def test_norm_against_fp64(comm, name, gt, layout):
    counts = LISTS[name]
    _, _, _, (g,) = _make(counts, 6, gt)
    # what lies between the tensors would make the norm inf
    gs = _aligned(g, TYPES[gt]) if layout == "aligned" else _views(g, TYPES[gt], 3, 0 if layout == "packed" else 5, math.inf)[1]
    n = _norm64(g, 0.5)
    for max_norm in (0.0, n / 3, n * 3):
        out = torch.full((2,), -1.0, device="cuda")
        comm.grad_norm_scattered(gs, out, max_norm=max_norm, grad_scale=-0.5)
        got = out.double().cpu().numpy()
        # fp32 sums of at most 8 squares: each 8 roundings at most, halved by the root, one on the way out
        assert abs(got[0] - n) <= 5.1 * A.U * n + 2.0 ** -149, (got, n)
        f32_max = float(np.float32(max_norm))
        clip = f32_max / n if 0 < f32_max < n else 1.0
        assert abs(got[1] - clip) <= 6.1 * A.U * clip
        again = torch.zeros(2, device="cuda")
        comm.grad_norm_scattered(gs, again, max_norm=max_norm, grad_scale=-0.5)
        assert torch.equal(again, out)


@pytest.mark.parametrize("values,expect", [
    ([0.0] * 1000, 0.0), ([1e-30] * 1000, None), ([2.0 ** -149] * 64, None), ([3e30] * 5 + [0.0] * 3000, None),
    ([3e38] * 4, math.inf), ([1.0, math.inf], math.inf), ([1.0, -math.inf, 2.0], math.inf), ([math.nan] + [1.0] * 600, math.nan),
    ([1e-25] * 7 + [1.0] + [1e20], None)])
@pytest.mark.parametrize("offset", [0, 1])
def test_norm_at_the_ends_of_the_range(comm, values, expect, offset):
    g = np.array(values, np.float32)
    out = torch.zeros(2, device="cuda")
    comm.grad_norm_scattered(_views([g], torch.float32, offset, 0)[1], out, max_norm=1.0)
    got = out.cpu().numpy().astype(np.float64)
    if expect is None:
        expect = _norm64([g])
        assert abs(got[0] - expect) <= 5.1 * A.U * expect + 2.0 ** -149
        clip = 1.0 / expect if expect > 1 else 1.0
        assert abs(got[1] - clip) <= 6.1 * A.U * clip
    else:
        assert got[0] == expect or (math.isnan(expect) and math.isnan(got[0]))
        assert got[1] == (1.0 if expect == 0.0 else 0.0)


@pytest.mark.parametrize("R", [2, 3, 8])
@pytest.mark.parametrize("gt", ["f32", "bf16"])
@pytest.mark.parametrize("packed", [False, True])
def test_norm_over_ranks(R, gt, packed):
    comms = coco.Communicator.init_all(R, [0] * R)
    try:
        for counts in (RAGGED, [1], [0, 0], [50001, 3]):
            _, _, _, g = _make(counts, 7, gt, ranks=R)
            outs = [torch.full((2,), -1.0, device="cuda") for _ in range(R)]
            gs = [_views(g[r], TYPES[gt], 1, 0)[1] if packed else _aligned(g[r], TYPES[gt]) for r in range(R)]
            with coco.group():
                for r, c in enumerate(comms):
                    c.grad_norm_scattered(gs[r], outs[r], max_norm=0.01)
            torch.cuda.synchronize()
            n = _norm64([A.sum32([g[r][b] for r in range(R)]) for b in range(len(counts))])
            for r, c in enumerate(comms):
                assert c.status()["code"] == 0
                assert torch.equal(outs[r], outs[0])
            assert abs(float(outs[0][0]) - n) <= 1.1 * A.U * n + 2.0 ** -149   # summed in fp64, rounded once
    finally:
        for c in comms:
            c.destroy()


# ---- used together, and from captured graphs ---------------------------------------
def _training(comm_calls, counts, steps, quant, capture=False):
    """Three steps of norm + AdamW on one GPU; returns weights, state, norms."""
    comm = comm_calls
    w, _, _, _ = _make(counts, 30, "bf16", step=0)
    ws = _aligned(w, torch.float32)
    gs = [torch.zeros(c, dtype=torch.bfloat16, device="cuda") for c in counts]
    lps = [x.bfloat16() for x in ws]
    lst = coco.TensorList(gs, ws, lps=lps, no_decay=[c < 100 for c in counts])
    state = coco.quant_state(counts, 1) if quant else tuple(torch.zeros(coco.scattered_slice_elems(counts, 1), device="cuda") for _ in range(2))
    norm, norms = torch.zeros(2, device="cuda"), []

    def step(k):
        comm.grad_norm_scattered(lst, norm, max_norm=0.02)
        if quant:
            comm.fused_adamw_quant_scattered(lst, None, *state, H["lr"], H["beta1"], H["beta2"], H["eps"], H["weight_decay"], k, 5, norm=norm)
        else:
            comm.fused_adamw_scattered(lst, None, *state, H["lr"], H["beta1"], H["beta2"], H["eps"], H["weight_decay"], k, norm=norm)

    for k in range(steps):
        _, _, _, (g,) = _make(counts, 40 + k, "bf16")
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
        norms.append(norm.clone())
    return ws, lps, state, norms


@pytest.mark.parametrize("quant", [False, True])
def test_steps_together_and_from_captured_graphs(comm, quant):
    counts = RAGGED
    ws, lps, state, norms = _training(comm, counts, 3, quant)
    cw, cl, cs, cn = _training(comm, counts, 3, quant, capture=True)
    assert all(torch.equal(a, b) for a, b in zip(ws + lps + norms, cw + cl + cn))
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(state, cs))
    # the same three steps in fp64, with each step's norm as it was returned
    w, _, _, _ = _make(counts, 30, "bf16", step=0)
    for b, c in enumerate(counts):
        x, m, v = w[b].astype(np.float64), np.zeros(c), np.zeros(c)
        slack = np.zeros(c)
        for k in range(3):
            _, _, _, (g,) = _make(counts, 40 + k, "bf16")
            n, clip = (float(y) for y in norms[k])
            assert abs(n - _norm64(g)) <= 5.1 * A.U * n
            x, m, v, q = A.step64(x, m, v, g[b].astype(np.float64) * clip, k, c >= 100)
            slack += 64 * A.U * (np.abs(x) + np.abs(q)) + 1e-12
        got = ws[b].cpu().numpy().astype(np.float64)
        if quant:   # the moments of the step before enter with a code step's relative error, 1/8, each
            slack += 3 * float(A.HYPER["lr"])
        assert (np.abs(got - x) <= slack).all(), b
        assert np.array_equal(lps[b].float().cpu().numpy(), ws[b].bfloat16().float().cpu().numpy())


def test_two_graphs_of_one_communicator_replay_in_any_order(comm):
    lists, outs, graphs = [], [], []
    for k in range(2):
        _, _, _, (g,) = _make([200003, 17, 5000 + k], 50 + k, "f32")
        lists.append(coco.TensorList(_aligned(g, torch.float32), None))
        outs.append(torch.zeros(2, device="cuda"))
        comm.grad_norm_scattered(lists[k], outs[k])
    torch.cuda.synchronize()
    expect = [o.clone() for o in outs]
    for k in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[k]):
            comm.grad_norm_scattered(lists[k], outs[k])
    for order in ((0, 1), (1, 0), (1, 1, 0)):
        for o in outs:
            o.zero_()
        for k in order:
            graphs[k].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], expect[0]) and torch.equal(outs[1], expect[1])


@pytest.mark.parametrize("op", ["norm", "adamw", "quant"])
def test_the_first_call_of_a_process_may_be_captured(op):
    """A list of two launches, captured before anything of the library has run; the replay against a plain call."""
    code = f"""
import torch, coconet_b200 as coco
comm = coco.Communicator.init_all(1, [0])[0]
counts = [1 + (k * 37) % 500 for k in range(1100)]
g = [torch.randn(c, device='cuda').bfloat16() for c in counts]
w = [torch.randn(c, device='cuda') for c in counts]
op = {op!r}
def state():
    if op == 'norm':
        return (torch.zeros(2, device='cuda'),)
    if op == 'quant':
        return coco.quant_state(counts, 1)
    return tuple(torch.zeros(coco.scattered_slice_elems(counts, 1), device='cuda') for _ in range(2))
def call(lst, st):
    if op == 'norm':
        comm.grad_norm_scattered(lst, *st)
    elif op == 'quant':
        comm.fused_adamw_quant_scattered(lst, None, *st, 1e-3, 0.9, 0.99, 1e-8, 0.1, 2, 3)
    else:
        comm.fused_adamw_scattered(lst, None, *st, 1e-3, 0.9, 0.99, 1e-8, 0.1, 2)
ws = [[x.clone() for x in w] for _ in range(2)]
sts = [state() for _ in range(2)]
lists = [coco.TensorList(g, x) for x in ws]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    call(lists[0], sts[0])
assert all(torch.equal(a, b) for a, b in zip(ws[0], w))
graph.replay()
call(lists[1], sts[1])
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(*ws))
assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(*sts))
assert op != 'norm' or float(sts[0][0][0]) > 0
assert op == 'norm' or not torch.equal(ws[0][1], w[1])
assert comm.launch_count() == 4 and comm.status()['code'] == 0
"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_calls_on_two_streams_do_not_disturb_each_other(comm):
    """AdamW calls at world size 1 share nothing: two lists stepped on two streams at once, ten times."""
    counts = [400003, 5, 70000]
    w, m, v, (g,) = _make(counts, 70, "f32")
    streams = [torch.cuda.Stream() for _ in range(2)]
    sets = []
    for _ in range(3):
        sets.append((coco.TensorList(_aligned(g, torch.float32), _aligned(w, torch.float32)),
                     [torch.from_numpy(_flat(x, counts, 8)).cuda() for x in (m, v)],
                     coco.TensorList(_aligned(g, torch.float32), _aligned(w, torch.float32)), coco.quant_state(counts, 1)))
    torch.cuda.synchronize()
    for k in range(10):
        for lst, st, qlst, qst in sets[:1]:
            comm.fused_adamw_scattered(lst, None, *st, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.1, k)
            comm.fused_adamw_quant_scattered(qlst, None, *qst, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.1, k, 1)
        for stream, (lst, st, qlst, qst) in zip(streams, sets[1:]):
            comm.fused_adamw_scattered(lst, None, *st, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.1, k, stream=stream)
            comm.fused_adamw_quant_scattered(qlst, None, *qst, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.1, k, 1, stream=stream)
    torch.cuda.synchronize()
    flat = [list(s[0].tensors[1]) + list(s[1]) + list(s[2].tensors[1]) + [x.view(torch.uint8) for x in s[3]] for s in sets]
    for other in flat[1:]:
        assert all(torch.equal(a, b) for a, b in zip(flat[0], other))


def test_another_stream_and_a_group_of_one(comm):
    counts = RAGGED
    w, m, v, (g,) = _make(counts, 60, "f32")
    results = []
    for how in ("plain", "stream", "group"):
        ws, gs = _aligned(w, torch.float32), _aligned(g, torch.float32)
        st = [torch.from_numpy(_flat(x, counts, 8)).cuda() for x in (m, v)]
        args = (gs, ws, *st, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.1, 3)
        torch.cuda.synchronize()
        if how == "plain":
            comm.fused_adamw_scattered(*args)
        elif how == "stream":
            s = torch.cuda.Stream()
            comm.fused_adamw_scattered(*args, stream=s)
            s.synchronize()
        else:
            with coco.group():
                comm.fused_adamw_scattered(*args)
        torch.cuda.synchronize()
        results.append(ws + st)
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))


def test_empty_lists_and_empty_tensors(comm):
    e, f = torch.zeros(0, device="cuda"), torch.zeros(4, device="cuda")
    out = torch.full((2,), -1.0, device="cuda")
    comm.grad_norm_scattered([e, e], out, max_norm=1.0)
    assert out.tolist() == [0.0, 1.0]
    comm.fused_adamw_scattered([e], [e.clone()], f, f.clone(), 1e-3, 0.9, 0.999, 1e-8, 0.0, 0)
    m, r, s = coco.quant_state([0], 1)
    comm.fused_adamw_quant_scattered([e], [e.clone()], m, r, s, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, 0)
    torch.cuda.synchronize()
    assert not f.any()


def test_refusals(comm):
    import ctypes as C
    L = coco.lib()
    n = 64
    t = {k: torch.ones(n, device="cuda") for k in "gwmv"}
    lp = torch.ones(n, dtype=torch.bfloat16, device="cuda")

    def call(counts=(n,), g=None, w=None, m=None, v=None, lp_ptr=None, lpt=9, gt=7, lr=1e-3, b1=0.9, b2=0.999,
             eps=1e-8, wd=0.0, step=0, gs=1.0, nbuff=1, norm=None):
        p = lambda k, x: t[k].data_ptr() if x is None else x  # noqa: E731
        one = lambda x: (C.c_void_p * 1)(x)                    # noqa: E731
        return L.cocoFusedAdamWScattered(comm._h, nbuff, one(p("g", g)), gt, one(p("w", w)),
                                         one(lp_ptr) if lp_ptr is not None else None, lpt, (C.c_size_t * 1)(*counts),
                                         p("m", m), p("v", v), lr, b1, b2, eps, wd, None, step, gs, norm, None)
    bad = [dict(nbuff=0), dict(gt=3), dict(lp_ptr=lp.data_ptr(), lpt=7), dict(lp_ptr=lp.data_ptr() + 1), dict(step=-1),
           dict(b1=1.0), dict(b2=1.0), dict(b1=-0.1), dict(b2=math.nan), dict(eps=-1e-8), dict(eps=math.nan), dict(eps=math.inf),
           dict(eps=1e-40), dict(lr=math.nan), dict(wd=math.inf), dict(gs=math.nan), dict(g=t["g"].data_ptr() + 2), dict(w=t["w"].data_ptr() + 1),
           dict(m=t["m"].data_ptr() + 2), dict(v=0), dict(m=0), dict(g=0), dict(w=0), dict(norm=t["v"].data_ptr() + 1),
           dict(counts=(1 << 40,))]
    for kw in bad:
        assert call(**kw) == 1, kw
    torch.cuda.synchronize()
    assert all(bool((x == 1).all()) for x in t.values())
    one = lambda x: (C.c_void_p * 1)(x)  # noqa: E731
    cnt = (C.c_size_t * 1)(n)
    norm = torch.zeros(4, device="cuda")
    for g, gt, out, scale, mx in [(t["g"].data_ptr(), 3, norm.data_ptr(), 1.0, 0.0), (t["g"].data_ptr() + 1, 7, norm.data_ptr(), 1.0, 0.0),
                                  (t["g"].data_ptr(), 7, 0, 1.0, 0.0), (t["g"].data_ptr(), 7, norm.data_ptr() + 2, 1.0, 0.0),
                                  (t["g"].data_ptr(), 7, norm.data_ptr(), math.nan, 0.0), (t["g"].data_ptr(), 7, norm.data_ptr(), 1.0, math.nan)]:
        assert L.cocoGradNormScattered(comm._h, 1, one(g), gt, cnt, scale, mx, out, None) == 1
    st = coco.quant_state([n], 1)
    q = lambda m, r, s, seed=0: L.cocoFusedAdamWQuantScattered(  # noqa: E731
        comm._h, 1, one(t["g"].data_ptr()), 7, one(t["w"].data_ptr()), None, 6, cnt, m, r, s, 1e-3, 0.9, 0.999, 1e-8, 0.0,
        None, 0, seed, 1.0, None, None)
    p = [x.data_ptr() for x in st]
    assert q(0, p[1], p[2]) == 1 and q(p[0], 0, p[2]) == 1 and q(p[0], p[1], 0) == 1 and q(p[0], p[1], p[2] + 1) == 1
    # the Python layer's own checks
    g, w, m, v = (t[k] for k in "gwmv")
    for args in [([g], [w.half()], m, v), ([g, g.half()], [w, w], m, v), ([g], [w], m[:32], v), ([g], [w], m.half(), v),
                 ([g[::2]], [w[:32]], m, v), ([g], [w[:32]], m, v), ([g], [w.cpu()], m, v), ([g.cpu()], [w.cpu()], m, v)]:
        with pytest.raises(ValueError):
            comm.fused_adamw_scattered(*args, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0)
    with pytest.raises(ValueError):
        comm.fused_adamw_scattered(coco.TensorList([g], None), None, m, v, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0)
    with pytest.raises(ValueError):
        comm.fused_adamw_scattered([g], [w], m, v, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, norm=torch.zeros(1, device="cuda"))
    with pytest.raises(ValueError):
        comm.fused_adamw_quant_scattered([g], [w], m, v, st[2], 1e-3, 0.9, 0.999, 1e-8, 0.0, 0, 0)
    with pytest.raises(coco.CocoError):
        comm.fused_adamw_scattered([g], [w], m, v, 1e-3, 1.5, 0.999, 1e-8, 0.0, 0)


def test_capture_is_refused_above_one_rank():
    comms = coco.Communicator.init_all(2, [0, 0])
    try:
        g, out = torch.ones(64, device="cuda"), torch.zeros(2, device="cuda")
        graph = torch.cuda.CUDAGraph()
        x = torch.zeros(4, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            x.add_(1.0)
            with pytest.raises(coco.CocoError) as e:
                comms[0].grad_norm_scattered([g], out)
            assert e.value.code == 2
        with coco.group():   # and the communicator is as usable as before
            for c in comms:
                c.grad_norm_scattered([g], out)
        torch.cuda.synchronize()
        assert out.tolist() == [16.0, 1.0]
    finally:
        for c in comms:
            c.destroy()


@pytest.mark.parametrize("op", ["adamw", "quant", "norm"])
def test_places_beyond_32_bits(comm, op):
    """A tensor of 2^32 + 300 elements behind a short one: its last elements, the first, and one in between."""
    n = (1 << 32) + 300
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 90 << 30:
        pytest.skip("needs 90 GB of free device memory")
    probe = [0, 1 << 20, (1 << 32) - 1, 1 << 32, n - 2, n - 1]
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    vals = torch.tensor([0.5, -1.0, 2.0, -0.25, 1.5, 3.0])
    g[torch.tensor(probe, device="cuda")] = vals.bfloat16().cuda()
    small = torch.zeros(9, dtype=torch.bfloat16, device="cuda")
    if op == "norm":
        out = torch.zeros(2, device="cuda")
        comm.grad_norm_scattered([small, g], out)
        n64 = math.sqrt(float((vals.double() ** 2).sum()))
        assert abs(float(out[0]) - n64) <= 5.1 * A.U * n64
        return
    counts = [9, n]
    w = torch.zeros(n, device="cuda")
    ws = [torch.zeros(9, device="cuda"), w]
    at = torch.tensor(probe, device="cuda")
    h = dict(lr=H["lr"], b1=H["beta1"], b2=H["beta2"], eps=H["eps"])
    if op == "adamw":
        m, v = (torch.zeros(coco.scattered_slice_elems(counts, 1), device="cuda") for _ in range(2))
        comm.fused_adamw_scattered([small, g], ws, m, v, *h.values(), 0.0, 0)
        rw, rm, rv = A.step32(np.zeros(6, np.float32), np.zeros(6, np.float32), np.zeros(6, np.float32), vals.numpy(), 0,
                              hyper=dict(A.HYPER, weight_decay=0.0))
        off = coco.scattered_tensor_place(counts, 1, 1)[0]
        assert np.array_equal(m[at + off].cpu().numpy(), rm) and np.array_equal(v[at + off].cpu().numpy(), rv)
        assert int((m != 0).sum()) == 6
    else:
        st = coco.quant_state(counts, 1)
        comm.fused_adamw_quant_scattered([small, g], ws, *st, *h.values(), 0.0, 0, 3)
        off = coco.quant_tensor_place(counts, 1, 1)[0]
        rw = np.empty(6, np.float32)
        for k, p in enumerate(probe):
            a = p // 256 * 256
            b = min(n, a + 256)
            z = np.zeros(b - a, np.float32)
            out = A.quant_step32(z, z.astype(np.uint8), z.astype(np.uint8), np.zeros((1, 2), np.uint8),
                                 g[a:b].float().cpu().numpy(), 0, 3, off + a, hyper=dict(A.HYPER, weight_decay=0.0))
            rw[k] = out[0][p - a]
            assert np.array_equal(st[0].view(torch.uint8)[off + a:off + b].cpu().numpy(), out[1]), p
            assert np.array_equal(st[1].view(torch.uint8)[off + a:off + b].cpu().numpy(), out[2]), p
            assert np.array_equal(st[2].view(torch.uint8)[(off + a) // 256].cpu().numpy(), out[3][0]), p
    assert (np.abs(w[at].cpu().numpy() - rw) <= 10 * A.U * np.abs(rw)).all()   # w = -q: near32
    assert int((w != 0).sum()) == 6


def test_a_norm_longer_than_a_launch_counts(comm):
    """2^31 groups of 16 bytes are one launch; the tensor ends 25 groups behind."""
    torch.cuda.empty_cache()
    n = (1 << 33) + 99
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    g = torch.zeros(n, device="cuda")
    for at, x in ((0, 1.0), ((1 << 33) - 1, 2.0), (1 << 33, 4.0), (n - 1, 8.0)):
        g[at] = x
    out, before = torch.zeros(2, device="cuda"), comm.launch_count()
    comm.grad_norm_scattered([g], out)
    assert comm.launch_count() == before + 2
    assert abs(float(out[0]) - math.sqrt(85.0)) <= 5.1 * A.U * math.sqrt(85.0)


@pytest.mark.parametrize("hyper", [
    dict(beta1=0.0, beta2=0.0), dict(beta1=0.5, beta2=0.125), dict(beta1=0.99, beta2=0.99999), dict(eps=0.0), dict(lr=0.0),
    dict(weight_decay=0.0, eps=1e-8), dict(beta1=0.0, beta2=0.999, eps=1.0)])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -44])
def test_hyper_parameters_at_their_ends(comm, hyper, scale):
    """Moments and codes bit for bit, weights near, for betas of 0 and near 1, no eps, no lr, and for gradients whose
    squares lie below the fp32 normal range."""
    h = {k: A.F(v) for k, v in dict(A.HYPER, **hyper).items()}
    n = 3000
    r = np.random.default_rng(11)
    g = (r.normal(0, 1e-3, n) * scale).astype(np.float32)
    g[g == 0] = np.float32(1e-3 * scale)
    w0 = r.normal(0, 0.02, n).astype(np.float32)
    args = [float(h[k]) for k in ("lr", "beta1", "beta2", "eps", "weight_decay")]
    gd = torch.from_numpy(g).cuda()
    w, m, v = torch.from_numpy(w0.copy()).cuda(), torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    q, st = torch.from_numpy(w0.copy()).cuda(), coco.quant_state([n], 1)
    om, ov, ow = np.zeros(n, np.float32), np.zeros(n, np.float32), w0.copy()
    mc, rc, sc = np.zeros(n, np.uint8), np.zeros(n, np.uint8), np.zeros((12, 2), np.uint8)
    for step in range(3):
        comm.fused_adamw_scattered([gd], [w], m, v, *args, step)
        comm.fused_adamw_quant_scattered([gd], [q], *st, *args, step, 4)
        before = (ow, om, ov, g)
        _, om, ov = A.step32(*before, step, hyper=h)
        assert np.array_equal(m.cpu().numpy(), om) and np.array_equal(v.cpu().numpy(), ov), step
        ow = w.cpu().numpy().copy()
        if scale == 1.0:   # (below, the root of a number without a normal range has no relative bound)
            assert A.near32(ow, *before, step, hyper=h), step
        out = A.quant_step32(w0, mc, rc, sc, g, step, 4, 0, hyper=h)
        _, mc, rc, sc = out[:4]
        assert np.array_equal(st[0].view(torch.uint8).cpu().numpy()[:n], mc), step
        assert np.array_equal(st[1].view(torch.uint8).cpu().numpy()[:n], rc), step
        assert np.array_equal(st[2].view(torch.uint8).cpu().numpy(), sc), step
        assert bool(torch.isfinite(q).all()), step


def test_fewer_ctas_give_the_same_step(comm):
    counts = RAGGED + [300001]
    w, m, v, (g,) = _make(counts, 80, "bf16")
    results = []
    for ctas in (0, 1):
        comm.set_tunables(ctas_per_sm=ctas)
        gs, ws, qs = _aligned(g, torch.bfloat16), _aligned(w, torch.float32), _views(w, torch.float32, 1, 0)[1]
        st, qst, norm = [torch.from_numpy(_flat(x, counts, 8)).cuda() for x in (m, v)], coco.quant_state(counts, 1), torch.zeros(2, device="cuda")
        comm.grad_norm_scattered(gs, norm, max_norm=0.01)
        assert abs(float(norm[0]) - _norm64(g)) <= 5.1 * A.U * _norm64(g)
        comm.fused_adamw_scattered(gs, ws, *st, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.1, 3)
        comm.fused_adamw_quant_scattered(gs, qs, *qst, H["lr"], H["beta1"], H["beta2"], H["eps"], 0.1, 3, 2)
        results.append(ws + qs + st + [x.view(torch.uint8) for x in qst])
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize("gt,lp", [("f32", "f16"), ("f16", "f16"), ("bf16", None)])
@pytest.mark.parametrize("packed", [False, True])
def test_quant_adamw_of_large_tensors_bit_for_bit(comm, gt, lp, packed):
    """Lists of 1024 and more units a tensor, on average, and of 8 tiles and more a CTA, with small tensors and ragged ends among them."""
    counts = [900001, 17, 5300000, 256, 40960 * 40]
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert sum(-(-c // 256) for c in counts) >= max(1024 * len(counts), 8 * 24 * sms)
    off, total = A.starts(counts, 256)[0], coco.quant_slice_elems(counts, 1)
    w, m, v, (g,) = _make(counts, 90, gt)
    state = _quant_initial(counts, m, v, 91)
    mf, rf, sf = np.full(total, 0x55, np.uint8), np.full(total, 0x55, np.uint8), np.full((total // 256, 2), 0x44, np.uint8)
    for o, (mc, rc, sc) in zip(off, state):
        mf[o:o + mc.size], rf[o:o + rc.size], sf[o // 256:o // 256 + len(sc)] = mc, rc, sc
    st = [torch.from_numpy(x.copy()).cuda() for x in (mf, rf, sf)]
    bufs = {}

    def place(name, arrays, dtype):
        if not packed:
            return _aligned(arrays, dtype)
        bufs[name] = _views(arrays, dtype, 1, 3)
        return bufs[name][1]
    gs, ws = place("g", g, TYPES[gt]), place("w", w, torch.float32)
    lps = place("lp", [np.zeros(c, np.float32) for c in counts], TYPES[lp]) if lp else None
    no_decay = [False, True, True, False, False]
    for step in (2, 3):
        comm.fused_adamw_quant_scattered(gs, ws, *st, H["lr"], H["beta1"], H["beta2"], H["eps"], H["weight_decay"], step, 77,
                                         w_lps=lps, no_decay=no_decay)
        gm, gr, gsc = (x.cpu().numpy() for x in st)
        for b, c in enumerate(counts):
            mc, rc, sc = state[b]
            old = (A.code_values(mc) * A.scale_values(sc[:, 0]).repeat(256)[:c],
                   (A.code_values(rc) * A.scale_values(sc[:, 1]).repeat(256)[:c]) ** 2)
            _, mc, rc, sc, _, _ = A.quant_step32(w[b], mc, rc, sc, g[b], step, 77, off[b], not no_decay[b])
            state[b] = (mc, rc, sc)
            assert np.array_equal(gm[off[b]:off[b] + c], mc), (step, b)
            assert np.array_equal(gr[off[b]:off[b] + c], rc), (step, b)
            assert np.array_equal(gsc[off[b] // 256:off[b] // 256 + len(sc)], sc), (step, b)
            before, now = w[b].astype(np.float64), ws[b].cpu().numpy()
            x = (before, old[0], old[1], g[b].astype(np.float64), step, not no_decay[b])
            assert (np.abs(now - A.step64(*x)[0]) <= A.bounds64(*x)[0]).all(), (step, b)
            w[b] = now
            if lp:
                assert np.array_equal(lps[b].float().cpu().numpy(), _lp_of(now, lp)), (step, b)
    assert all(_gaps_untouched(*x) for x in bufs.values())
    used = np.zeros(total, bool)
    for o, c in zip(off, counts):
        used[o:o + c] = True
    gm, gr, _ = (x.cpu().numpy() for x in st)
    assert (gm[~used] == 0x55).all() and (gr[~used] == 0x55).all()
