"""Plain evaluations of AdamW and its 8-bit state for the tests: in fp64 from the
definition, and in fp32 with every operation rounded by itself, which the
kernels' moments, codes and scales have to match bit for bit.  The weights, whose
update goes through the hardware's reciprocal and root, have to match it within
`near32`.  numpy only."""
import math

import numpy as np

BLOCK = 256
F = np.float32
U = 2.0 ** -24   # half a step of fp32, relative

HYPER = dict(lr=F(1e-3), beta1=F(0.9), beta2=F(0.999), eps=F(1e-6), weight_decay=F(0.01))


def starts(counts, align):
    at, out = 0, []
    for c in counts:
        out.append(at)
        at += -(-c // align) * align
    return out, at


def slice_elems(counts, world, align):
    total = starts(counts, align)[1]
    return -(-(-(-total // world)) // align) * align


# ---- fp64 -----------------------------------------------------------------------
def step64(w, m, v, g, step, decays=True, lr=None, beta1=None, beta2=None, eps=None, weight_decay=None):
    """One step on arrays of doubles: new (w, m, v), and the update q that w lost."""
    h = {k: float(x) for k, x in HYPER.items()}
    h.update({k: float(x) for k, x in dict(lr=lr, beta1=beta1, beta2=beta2, eps=eps, weight_decay=weight_decay).items()
              if x is not None})
    t = step + 1
    m = h["beta1"] * m + (1 - h["beta1"]) * g
    v = h["beta2"] * v + (1 - h["beta2"]) * g * g
    q = h["lr"] * (m / (1 - h["beta1"] ** t)) / (np.sqrt(v / (1 - h["beta2"] ** t)) + h["eps"])
    w = w * (1 - h["lr"] * h["weight_decay"] if decays else 1.0) - q
    return w, m, v, q


def bounds64(w, m, v, g, step, decays=True):
    """How far fp32 results may be from step64's, from the roundings on the way (u = 2^-24):
      g'  = g s                                   1 rounding
      m'  = (m b1) + (g' omb1)                    u (2 |m b1| + 3 |g omb1|)
      v'  = (v b2) + ((g' g') omb2)               at most 5 roundings of its larger part, no cancellation
      r   = sqrt(v'), den = r rs2 + eps           2.5 + 2 (the hardware's root: 2^-23), + 1 (rs2) + 1 + 1: 7.5 u
      q   = (m' c1) * (1 / den)                   m' error / m' + 1 (c1) + 1 + 2 (its reciprocal) + 1 + 7.5 u
      w'  = w decay - q                           2 u |w| + error of q + u |w'|
    and 2^-140 for what the smallest numbers lose below the normal range (six places of at most 2^-149)."""
    b1, b2 = float(HYPER["beta1"]), float(HYPER["beta2"])
    w1, m1, v1, q = step64(w, m, v, g, step, decays)
    tiny = 2.0 ** -140
    em = 1.01 * U * (2 * np.abs(m * b1) + 3 * np.abs(g * (1 - b1))) + tiny
    ev = 1.01 * U * 5 * v1 + tiny
    with np.errstate(divide="ignore", invalid="ignore"):
        per_m = np.where(m1 != 0, np.abs(q / np.where(m1 != 0, m1, 1)), 0.0)  # dq / dm
    per_m = np.where(m1 != 0, per_m, float(HYPER["lr"]) / (1 - b1 ** (step + 1)) /
                     (np.sqrt(v1 / (1 - b2 ** (step + 1))) + float(HYPER["eps"])))
    eq = em * per_m + 1.01 * U * 12.5 * np.abs(q) + tiny
    ew = 1.01 * U * (2 * np.abs(w) + np.abs(w1)) + eq + tiny
    return ew, em, ev


# ---- fp32, operation by operation ------------------------------------------------
def scalars32(step, lr, beta1, beta2, eps, weight_decay):
    d1 = 1.0 - math.pow(float(beta1), step + 1.0)
    d2 = 1.0 - math.pow(float(beta2), step + 1.0)
    return dict(b1=F(beta1), b2=F(beta2), omb1=F(1) - F(beta1), omb2=F(1) - F(beta2), eps=F(eps),
                c1=F(float(lr) / d1), rs2=F(1.0 / math.sqrt(d2)), decay=F(1.0 - float(lr) * float(weight_decay)))


def moments32(h, m, v, g):
    return m * h["b1"] + g * h["omb1"], v * h["b2"] + (g * g) * h["omb2"]


def weights32(h, w, m, r, decays):
    return w * (h["decay"] if decays else F(1)) - (m * h["c1"]) / (r * h["rs2"] + h["eps"])


def factor32(grad_scale, norm):
    return F(grad_scale) if norm is None else F(norm[1]) * F(grad_scale)


def sum32(grads):
    """Sum over ranks in rank order in fp32 (the gradients are fp32 or were widened exactly)."""
    x = grads[0].astype(F)
    for g in grads[1:]:
        x = x + g.astype(F)
    return x


def near32(got, w, m, v, g, step, decays=True, hyper=HYPER):
    """Whether the weights `got` are step32's up to the two approximations: w - q with q off by
    2 u (root) + 2 u (reciprocal) and, as the operations before and after round differently, 4 u more; and the
    last subtraction half a step of either side.  (m, v, w, g: before the step.)"""
    w1, m1, v1 = step32(w, m, v, g, step, decays, hyper)
    with np.errstate(all="ignore"):
        h = scalars32(step, **hyper)
        q = np.abs((m1 * h["c1"]) / (np.sqrt(v1) * h["rs2"] + h["eps"])).astype(np.float64)
        far = np.abs(got.astype(np.float64) - w1.astype(np.float64))
        return bool((far <= 8 * U * q + 2 * U * np.abs(w1.astype(np.float64)) + 2.0 ** -140).all())


def step32(w, m, v, g, step, decays=True, hyper=HYPER):
    with np.errstate(all="ignore"):
        h = scalars32(step, **hyper)
        m, v = moments32(h, m, v, g)
        return weights32(h, w, m, np.sqrt(v), decays), m, v


# ---- 8-bit state -----------------------------------------------------------------
_M = np.uint64(0xFFFFFFFF)


def mix(x):
    x = np.asarray(x, np.uint64)
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x6A09E667)) & _M
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0xBB67AE85)) & _M
    return x ^ (x >> np.uint64(16))


def rounding_bits(first, n, seed, step):
    """32 random bits for every element of the flat state from `first` on."""
    with np.errstate(over="ignore"):
        key = mix((mix(seed & 0xFFFFFFFF) + np.uint64(seed >> 32) * np.uint64(0x3C6EF373) +
                   np.uint64(step) * np.uint64(0x9E3779B1)) & _M)
        f = np.uint64(first) + np.arange(n, dtype=np.uint64)
        return mix(((f & _M) * np.uint64(0x9E3779B1) + (f >> np.uint64(32)) * np.uint64(0x3C6EF373) + key) & _M).astype(np.uint32)


def code_values(codes):
    """e4m3 code bytes as doubles."""
    codes = np.asarray(codes, np.uint8)
    e, f = (codes >> 3) & 15, (codes & 7).astype(np.float64)
    x = np.where(e == 0, f * 2.0 ** -9, (1 + f / 8) * np.exp2(e.astype(np.float64) - 7))
    return np.where(codes & 0x80, -x, x)


def scale_values(scale):
    return np.where(scale == 255, np.nan, np.exp2(scale.astype(np.float64) - 127))


def encode32(x, bits16):
    """(codes, scale byte) of one tensor's values x; its last block may be short."""
    codes = np.empty(x.size, np.uint8)
    scales = np.empty(-(-x.size // BLOCK), np.uint8)
    with np.errstate(all="ignore"):
        for b in range(scales.size):
            y, r = x[b * BLOCK:(b + 1) * BLOCK], bits16[b * BLOCK:(b + 1) * BLOCK].astype(np.uint32)
            top = int((y.view(np.uint32) & np.uint32(0x7FFFFFFF)).max())
            if top >= 0x7F800000:
                codes[b * BLOCK:(b + 1) * BLOCK], scales[b] = 0, 255
                continue
            e = min(max(top >> 23, 8), 254)
            inv = np.array([(261 - e) << 23], np.uint32).view(F)[0]
            z = (np.abs(y) * inv) * F(2.0 ** -120)
            c = (z.view(np.uint32) + ((r << np.uint32(4)) | np.uint32(8))) >> np.uint32(20)
            codes[b * BLOCK:(b + 1) * BLOCK] = c | ((y.view(np.uint32) >> np.uint32(24)) & np.uint32(0x80))
            scales[b] = e - 7
    return codes, scales


def quant_step32(w, m_codes, r_codes, scales, g, step, seed, place, decays=True, hyper=HYPER):
    """One tensor: scales [blocks, 2]; `place`: its first element in the flat state.
    New (w, m codes, r codes, scales, m, r): the last two before rounding."""
    with np.errstate(all="ignore"):
        h = scalars32(step, **hyper)
        sc = scale_values(scales).astype(F).repeat(BLOCK, 0)[:w.size]
        m = code_values(m_codes).astype(F) * sc[:, 0]
        r = code_values(r_codes).astype(F) * sc[:, 1]
        m, v = moments32(h, m, r * r, g)
        r = np.sqrt(v)
        w = weights32(h, w, m, r, decays)
        bits = rounding_bits(place, w.size, seed, step)
        mc, ms = encode32(m, bits & np.uint32(0xFFFF))
        rc, rs = encode32(r, bits >> np.uint32(16))
        live = (r > 0) & (rs.repeat(BLOCK)[:w.size] != 255)
        rc = np.where(live & (rc == 0), np.uint8(1), rc)
    return w, mc, rc, np.stack([ms, rs], 1), m, r
