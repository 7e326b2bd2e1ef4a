"""The optimizer step of a large model, measured: AdamW over a list of tensors with 32-bit
moments, the same with moments held in 8 bits, and the global gradient norm with its clip factor.

Each is here in its plain form (elementary torch operations on flat buffers) and, where `own` is
true, as the call that a training program makes of this package.  A list of tensors is a set of
views into flat buffers, as in a program that keeps its gradients and weights in buckets, so that
the plain form can work on whole buffers.

The arithmetic, per element, with 32-bit hyper-parameters, t = step + 1, d1 = 1 - beta1^t,
d2 = 1 - beta2^t, s = grad_scale * clip factor:

    g  <- g * s
    m  <- beta1 * m + (1 - beta1) * g
    v  <- beta2 * v + (1 - beta2) * g^2
    w  <- w * (1 - lr * weight_decay) - (lr / d1 * m) / (sqrt(v) / sqrt(d2) + eps)

and the low-precision copy of w, where there is one, is w rounded.  A step whose gradient norm is
not finite changes nothing.

Moments in 8 bits: m and r = sqrt(v) are stored as e4m3 codes (8 bits: sign, 4 exponent, 3 mantissa
bits) times a power-of-two scale for every 256 elements, itself 8 bits (e8m0: the exponent of a 32-bit
float).  Every tensor starts a new block of the flat state.  With the block's largest absolute value in [2^e, 2^(e+1)) the scale is 2^(e-7), so that the
largest code lies in [128, 256); e is held at -119 or more.  A value is rounded up or down at random,
up with the probability of the part cut off, in units of 2^-20: 16 random bits, then a one, then
three zeros.  The random bits are a hash of the seed, the step and the element's place in the flat
state (`_hash`); the low half of the 32 bits serves m, the high half r.  An r above zero is
never stored as zero.
"""
import math
import random

import numpy as np
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BLOCK = 256  # elements of 8-bit state that share a scale
_M32 = 0xFFFFFFFF
_HYPER = {"lr": 1e-3, "beta1": 0.9, "beta2": 0.999, "eps": 1e-6, "weight_decay": 0.01}


# ---- lists of tensors ---------------------------------------------------------------------------
def _bert_large():
    """398 tensors, 336 M elements: 24 layers, hidden 1024, FFN 4096, vocabulary 30522, 512 positions."""
    sizes = [30522 * 1024, 512 * 1024, 2 * 1024, 1024, 1024]
    for _ in range(24):
        sizes += [1024 * 1024, 1024] * 4 + [1024, 1024]
        sizes += [1024 * 4096, 4096, 4096 * 1024, 1024, 1024, 1024]
    return sizes + [1024 * 1024, 1024, 1024 * 1024, 1024, 1024, 1024, 30522, 2 * 1024, 2]


def _counts(case):
    kind = case["list"]
    if kind == "bert-large":
        return _bert_large()
    if kind == "layer":  # one transformer layer
        h, f = case["hidden"], 4 * case["hidden"]
        return [h * h, h] * 4 + [h, h] + [h * f, f, f * h, h, h, h]
    # ragged: sizes spread over their logarithm, from one element on
    r = random.Random(case["sizes_seed"])
    return [max(1, int(math.exp(r.uniform(0.0, math.log(case["largest"] + 1))))) for _ in range(case["tensors"])]


def _starts(counts, align):
    at, starts = 0, []
    for c in counts:
        starts.append(at)
        at += -(-c // align) * align
    return starts, at


def listed():
    return [
        # the weight and bias of one normalisation, stepped by themselves: latency
        {"name": "adamw norm vectors", "op": "adamw", "list": "ragged", "tensors": 2, "largest": 1024, "sizes_seed": 1, "g": "f32", "lp": "none", "packed": False, "step": 100, "clip": False},
        # one layer of a mixed-precision run, from the first step, clipped
        {"name": "adamw one layer", "op": "adamw", "list": "layer", "hidden": 1024, "g": "bf16", "lp": "bf16", "packed": False, "step": 0, "clip": True},
        # a bucket without padding: nearly no tensor starts on a 16-byte boundary; many small tensors
        {"name": "adamw packed bucket", "op": "adamw", "list": "ragged", "tensors": 900, "largest": 400000, "sizes_seed": 2, "g": "f16", "lp": "f16", "packed": True, "step": 1000, "clip": True},
        # a whole model in 32 bits
        {"name": "adamw model fp32", "op": "adamw", "list": "bert-large", "g": "f32", "lp": "none", "packed": False, "step": 1000, "clip": False},
        # a whole model in mixed precision
        {"name": "adamw model bf16", "op": "adamw", "list": "bert-large", "g": "bf16", "lp": "bf16", "packed": False, "step": 1000, "clip": True},
        # the same four with 8-bit moments
        {"name": "adamw8 norm vectors", "op": "adamw8", "list": "ragged", "tensors": 2, "largest": 1024, "sizes_seed": 1, "g": "f32", "lp": "none", "packed": False, "step": 100, "clip": False},
        {"name": "adamw8 one layer", "op": "adamw8", "list": "layer", "hidden": 1024, "g": "bf16", "lp": "bf16", "packed": False, "step": 0, "clip": True},
        {"name": "adamw8 packed bucket", "op": "adamw8", "list": "ragged", "tensors": 900, "largest": 400000, "sizes_seed": 2, "g": "f16", "lp": "f16", "packed": True, "step": 1000, "clip": True},
        {"name": "adamw8 model bf16", "op": "adamw8", "list": "bert-large", "g": "bf16", "lp": "bf16", "packed": False, "step": 1000, "clip": True},
        # the norm that decides the clip factor: of a layer, of a packed bucket, of a whole model
        {"name": "norm one layer", "op": "norm", "list": "layer", "hidden": 1024, "g": "bf16", "packed": False},
        {"name": "norm packed bucket", "op": "norm", "list": "ragged", "tensors": 900, "largest": 400000, "sizes_seed": 2, "g": "f16", "packed": True},
        {"name": "norm model fp32", "op": "norm", "list": "bert-large", "g": "f32", "packed": False},
    ]


def draw(rng):
    op = rng.choice(["adamw", "adamw8", "norm"])
    tensors = int(math.exp(rng.uniform(0.0, math.log(1500.0))))
    # a list of n log-uniform sizes up to L holds about n * L / ln(L) elements: up to some 100 M
    most = max(4.0, min(8.0e7, 1.0e9 / tensors))
    case = {"op": op, "list": "ragged", "tensors": tensors, "largest": int(math.exp(rng.uniform(math.log(4.0), math.log(most)))),
            "sizes_seed": rng.randrange(1 << 30), "g": rng.choice(["f32", "f16", "bf16"]), "packed": rng.random() < 0.5}
    if op != "norm":
        case |= {"lp": rng.choice(["none", "f16", "bf16"]), "step": rng.choice([0, 1, rng.randrange(2, 100000)]), "clip": rng.random() < 0.5}
    return case


# ---- inputs -------------------------------------------------------------------------------------
def _inputs(case, seed):
    """What the program has in hand: views of flat buffers, the moments, the plain form's index maps."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    counts = _counts(case)
    starts, total = _starts(counts, 1 if case["packed"] else 8)
    gt = _DTYPES[case["g"]]
    scaled = case["g"] == "f16"  # a loss scale, as 16-bit gradients of a narrow range need
    s = {"op": case["op"], "counts": counts, "starts": starts, "grad_scale": 1.0 / 1024.0 if scaled else 1.0}

    tc = torch.tensor(counts, device=dev)
    ts = torch.tensor(starts, device=dev)
    tensor_of = torch.repeat_interleave(torch.arange(len(counts), device=dev), tc)
    inside = torch.arange(int(sum(counts)), device=dev) - (torch.cumsum(tc, 0) - tc)[tensor_of]
    place = ts[tensor_of] + inside  # of every element in the flat buffers

    def flat(values, dtype):
        if case["packed"]:
            return values.to(dtype)
        return torch.zeros(total, dtype=dtype, device=dev).index_copy_(0, place, values.to(dtype))

    n = place.numel()
    g = torch.randn(n, device=dev, generator=gen) * 1e-3
    g *= torch.rand(n, device=dev, generator=gen) > 0.1  # units that a batch does not reach
    s["g"] = flat(g * 1024.0 if scaled else g, gt)
    if case["op"] == "norm":
        s["max_norm"] = 1.0
        s["norm"] = torch.zeros(2, device=dev)
        return s

    s["w"] = flat(torch.randn(n, device=dev, generator=gen) * 0.02, torch.float32)
    s["lp"] = s["w"].to(_DTYPES[case["lp"]]) if case["lp"] != "none" else None
    s["norm"] = torch.tensor([2.5, 0.4], device=dev) if case["clip"] else None
    s["step"], s["seed"] = case["step"], seed & 0x7FFFFFFF
    s["no_decay"] = [c < 8192 for c in counts]  # biases and norms are not decayed
    decayed = torch.tensor([c >= 8192 for c in counts], device=dev)[tensor_of]
    s["decayed"] = decayed if case["packed"] else torch.zeros(total, dtype=torch.bool, device=dev).index_copy_(0, place, decayed)

    if case["step"] == 0:
        m, v = torch.zeros(n, device=dev), torch.zeros(n, device=dev)
    else:
        m = torch.randn(n, device=dev, generator=gen) * 3e-4
        v = torch.exp(torch.randn(n, device=dev, generator=gen)) * 1e-6
    align = 8 if case["op"] == "adamw" else _BLOCK
    state_starts, state_total = _starts(counts, align)
    state_place = torch.tensor(state_starts, device=dev)[tensor_of] + inside
    flat_m = torch.zeros(state_total, device=dev).index_copy_(0, state_place, m)
    flat_v = torch.zeros(state_total, device=dev).index_copy_(0, state_place, v)
    # where the plain form finds the state of the elements of the flat buffers: [buffer places], [state places]
    s["maps"] = None if align == 8 and not case["packed"] else (place, state_place)
    if case["op"] == "adamw":
        s["m"], s["v"] = flat_m, flat_v
        return s
    codes, scales = [], []
    for x in (flat_m, flat_v.sqrt_()):
        x = x.view(-1, _BLOCK)
        e = torch.floor(torch.log2(x.abs().amax(1).clamp_min(2.0 ** -119)))
        codes.append((x / torch.exp2(e - 7)[:, None]).to(torch.float8_e4m3fn).view(-1))
        scales.append((e + 120).to(torch.uint8))
    s["m"], s["r"] = codes
    s["scales"] = torch.stack(scales, 1).contiguous().view(torch.float8_e8m0fnu)
    return s


_comm = None


def _communicator():
    global _comm
    if _comm is None:
        import coconet_b200 as coco
        _comm = coco.Communicator.init_all(1)[0]
    return _comm


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:  # the communicator and the pointer lists that a training program makes once
        import coconet_b200 as coco
        s["comm"] = _communicator()
        views = [[flat[a:a + c] for a, c in zip(s["starts"], s["counts"])] if flat is not None else None
                 for flat in (s["g"], s.get("w"), s.get("lp"))]
        s["tensors"] = coco.TensorList(views[0], views[1], lps=views[2], no_decay=s.get("no_decay"))
    return s


# ---- the plain forms ----------------------------------------------------------------------------
def _scalars(step):
    """The hyper-parameters as 32-bit values, and what the step derives from them once."""
    f = np.float32
    lr, b1, b2, eps, wd = (f(_HYPER[k]) for k in ("lr", "beta1", "beta2", "eps", "weight_decay"))
    d1 = 1.0 - float(b1) ** (step + 1)
    d2 = 1.0 - float(b2) ** (step + 1)
    return {"b1": float(b1), "b2": float(b2), "omb1": float(f(1) - b1), "omb2": float(f(1) - b2), "eps": float(eps),
            "c1": float(f(float(lr) / d1)), "rs2": float(f(1.0 / math.sqrt(d2))), "decay": float(f(1.0 - float(lr) * float(wd)))}


def _gradient(s):
    """The scaled gradient in 32 bits, and whether the step is taken (None: always)."""
    g = s["g"].float()
    if s["norm"] is None:
        return g * s["grad_scale"], None
    return g * (s["norm"][1] * s["grad_scale"]), torch.isfinite(s["norm"][0])


def _moments(h, m, v, g):
    return m * h["b1"] + g * h["omb1"], v * h["b2"] + (g * g) * h["omb2"]


def _store(s, taken, **new):
    for k, x in new.items():
        s[k].copy_(x if taken is None else torch.where(taken, x, s[k]))


def _new_weights(h, s, update):
    w = torch.where(s["decayed"], s["w"] * h["decay"], s["w"]) - update
    return {"w": w} if s["lp"] is None else {"w": w, "lp": w.to(s["lp"].dtype)}


def _run_adamw(s):
    h = _scalars(s["step"])
    g, taken = _gradient(s)
    m, v = s["m"], s["v"]
    if s["maps"] is not None:
        place, state_place = s["maps"]
        g = torch.zeros_like(m).index_copy_(0, state_place, g)  # a packed buffer's places are 0, 1, ...
    m, v = _moments(h, m, v, g)
    update = (m * h["c1"]) / (torch.sqrt(v) * h["rs2"] + h["eps"])
    if s["maps"] is not None:
        update = update[state_place]
    _store(s, taken, m=m, v=v, **_new_weights(h, s, update))
    return {k: s[k] for k in ("w", "lp", "m", "v")}


def _hash(n, seed, step, device):
    """32 random bits for every place of the flat state, as a 64-bit tensor: multiply and xor-shift,
    the multipliers from the binary fractions of the golden ratio and the roots of 2, 3 and 5."""
    def mix(x):
        x = ((x ^ (x >> 16)) * 0x6A09E667) & _M32
        x = ((x ^ (x >> 15)) * 0xBB67AE85) & _M32
        return x ^ (x >> 16)
    key = mix((mix(seed & _M32) + (seed >> 32) * 0x3C6EF373 + step * 0x9E3779B1) & _M32)
    f = torch.arange(n, device=device)
    return mix(((f & _M32) * 0x9E3779B1 + (f >> 32) * 0x3C6EF373 + key) & _M32)


def _encode(x, bits16):
    """The codes and the blocks' scales of x [blocks, 256], as bytes in 32-bit integers."""
    e = (x.abs().amax(1).view(torch.int32) >> 23).clamp(8, 254)
    inverse = ((261 - e) << 23).view(torch.float32)
    y = (x.abs() * inverse[:, None]) * 2.0 ** -120  # the code's bits now lead the 32-bit float's
    code = (y.view(torch.int32) + ((bits16 << 4) | 8)) >> 20
    return code | ((x.view(torch.int32) >> 24) & 0x80), e - 7


def _run_adamw8(s):
    h = _scalars(s["step"])
    g, taken = _gradient(s)
    n = s["m"].numel()
    place, state_place = s["maps"]
    padded = torch.zeros(n, device=g.device).index_copy_(0, state_place, g[place])
    scales = s["scales"].float()
    m = s["m"].float().view(-1, _BLOCK) * scales[:, 0:1]
    r = s["r"].float().view(-1, _BLOCK) * scales[:, 1:2]
    m, v = _moments(h, m, r * r, padded.view(-1, _BLOCK))
    r = torch.sqrt(v)
    update = (m * h["c1"]) / (r * h["rs2"] + h["eps"])
    bits = _hash(n, s["seed"], s["step"], g.device).view(-1, _BLOCK)
    m_code, m_scale = _encode(m, (bits & 0xFFFF).to(torch.int32))
    r_code, r_scale = _encode(r, (bits >> 16).to(torch.int32))
    r_code = torch.where(r > 0, r_code.clamp_min(1), r_code)
    in_buffer = torch.zeros_like(s["w"]).index_copy_(0, place, update.view(-1)[state_place])
    _store(s, taken, **_new_weights(h, s, in_buffer))
    for k, code in (("m", m_code), ("r", r_code), ("scales", torch.stack([m_scale, r_scale], 1))):
        old = s[k].view(torch.uint8)
        code = code.to(torch.uint8).view(old.shape)
        old.copy_(code if taken is None else torch.where(taken, code, old))
    return {k: s[k] for k in ("w", "lp", "m", "r", "scales")}


def _run_norm(s):
    """In 64 bits: the sum runs over the whole model."""
    n = s["g"].double().square().sum().sqrt() * s["grad_scale"]
    clip = torch.where(n > s["max_norm"], s["max_norm"] / n, torch.ones_like(n))
    s["norm"].copy_(torch.stack([n, torch.where(torch.isfinite(n), clip, torch.zeros_like(n))]))
    return s["norm"]


def run(state):
    s = state
    if not own:
        return {"adamw": _run_adamw, "adamw8": _run_adamw8, "norm": _run_norm}[s["op"]](s)
    h = _HYPER
    if s["op"] == "norm":
        s["comm"].grad_norm_scattered(s["tensors"], s["norm"], max_norm=s["max_norm"], grad_scale=s["grad_scale"])
        return s["norm"]
    if s["op"] == "adamw":
        s["comm"].fused_adamw_scattered(s["tensors"], None, s["m"], s["v"], h["lr"], h["beta1"], h["beta2"], h["eps"],
                                        h["weight_decay"], s["step"], grad_scale=s["grad_scale"], norm=s["norm"])
        return {k: s[k] for k in ("w", "lp", "m", "v")}
    s["comm"].fused_adamw_quant_scattered(s["tensors"], None, s["m"], s["r"], s["scales"], h["lr"], h["beta1"], h["beta2"],
                                          h["eps"], h["weight_decay"], s["step"], s["seed"], grad_scale=s["grad_scale"],
                                          norm=s["norm"])
    # the e4m3 codes as the numbers they are, and beside them the scales that multiply every 256 of them
    return {k: s[k] for k in ("w", "lp", "m", "r", "scales")}


def work(case):
    n = sum(_counts(case))
    gb = 4 if case["g"] == "f32" else 2
    if case["op"] == "norm":
        return {"bytes": n * gb + 8, "flops": 2 * n}
    lp = 0 if case["lp"] == "none" else 2
    if case["op"] == "adamw":  # g; w, m, v read and written; the copy written
        return {"bytes": n * (gb + 24 + lp), "flops": 14 * n}
    blocks = sum(-(-c // _BLOCK) for c in _counts(case))
    return {"bytes": n * (gb + 8 + 4 + lp) + blocks * 4, "flops": 14 * n}


# ---- the definition in 64 bits -------------------------------------------------------------------
def exact(case, seed):
    s = _inputs(case, seed)
    dev = s["g"].device
    if s["op"] == "norm":
        total = sum(float((p.to(torch.float64) ** 2).sum()) for p in torch.split(s["g"], 1 << 26))
        n = math.sqrt(total) * s["grad_scale"]
        return torch.tensor([n, min(1.0, s["max_norm"] / n) if n > 0 else 1.0], dtype=torch.float64)
    p = {k: float(np.float32(v)) for k, v in _HYPER.items()}
    t = s["step"] + 1
    factor = s["grad_scale"] * (float(s["norm"][1]) if s["norm"] is not None else 1.0)
    counts, eight = s["counts"], s["op"] == "adamw8"
    state_starts, _ = _starts(counts, _BLOCK if eight else 8)
    w = s["w"].to(torch.float64)
    out = {"w": w, "lp": None}
    if eight:
        scales = s["scales"].to(torch.float64)
        m = s["m"].to(torch.float64) * scales[:, 0].repeat_interleave(_BLOCK)
        r = s["r"].to(torch.float64) * scales[:, 1].repeat_interleave(_BLOCK)
        v = r * r
    else:
        m, v = s["m"].to(torch.float64), s["v"].to(torch.float64)
    for a, b, c in zip(s["starts"], state_starts, counts):  # tensor by tensor, as the step is defined
        g = s["g"][a:a + c].to(torch.float64) * factor
        mt, vt, wt = m[b:b + c], v[b:b + c], w[a:a + c]
        mt.add_((g - mt) * (1 - p["beta1"]))
        vt.add_((g * g - vt) * (1 - p["beta2"]))
        if c >= 8192:
            wt.sub_(wt * (p["lr"] * p["weight_decay"]))
        wt.sub_(p["lr"] * (mt / (1 - p["beta1"] ** t)) / ((vt / (1 - p["beta2"] ** t)).sqrt() + p["eps"]))
    if s["lp"] is not None:
        out["lp"] = w.to(torch.float64)
    if not eight:
        return out | {"m": m, "v": v}
    bits = _hash(m.numel(), s["seed"], s["step"], dev)
    new_scales = []
    for name, x, u in (("m", m, bits & 0xFFFF), ("r", v.sqrt(), bits >> 16)):
        blocks = x.view(-1, _BLOCK)
        _, e = torch.frexp(blocks.abs().amax(1))  # in [0.5, 1) * 2^e
        scale = torch.ldexp(torch.ones_like(blocks[:, 0]), (e - 1).clamp(min=-119) - 7)
        y = blocks.abs() / scale[:, None]
        step = torch.ldexp(torch.ones_like(y), (torch.frexp(y)[1] - 1).clamp(min=-6) - 3)
        up = (u.view(-1, _BLOCK).to(torch.float64) * 16 + 8) / 2 ** 20
        q = torch.floor(y / step + up) * step
        if name == "r":
            q = torch.where((y > 0) & (q == 0), torch.full_like(q, 2.0 ** -9), q)
        out[name] = (q * torch.sign(blocks)).view(-1)
        new_scales.append(scale)
    return out | {"scales": torch.stack(new_scales, 1)}
