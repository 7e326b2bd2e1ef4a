"""AdamW and the gradient norm without a GPU: refusals that need no device, the
layout of the 8-bit state, and the tests' own evaluations against each other."""
import ctypes as C

import numpy as np
import pytest
import torch

import adamw_ref as A
import coconet_b200 as coco


def test_null_communicators_and_lists_are_refused():
    L = coco.lib()
    p, n = (C.c_void_p * 1)(64), (C.c_size_t * 1)(4)
    assert L.cocoGradNormScattered(None, 1, p, 7, n, 1.0, 0.0, 64, None) == 1
    assert L.cocoFusedAdamWScattered(None, 1, p, 7, p, None, 6, n, 64, 64, 1e-3, 0.9, 0.999, 1e-8, 0.0, None, 0, 1.0,
                                     None, None) == 1
    assert L.cocoFusedAdamWQuantScattered(None, 1, p, 7, p, None, 6, n, 64, 64, 64, 1e-3, 0.9, 0.999, 1e-8, 0.0, None, 0,
                                          0, 1.0, None, None) == 1
    out = C.c_size_t()
    assert L.cocoQuantSliceElems(1, None, 1, C.byref(out)) == 1
    assert L.cocoQuantSliceElems(1, n, 0, C.byref(out)) == 1
    assert L.cocoQuantSliceElems(1, n, 9, C.byref(out)) == 1


def test_python_checks_come_before_the_library():
    c = coco.Communicator(None, 1, 0)   # never reaches the library
    t = torch.zeros(16)
    with pytest.raises(ValueError, match="CUDA"):
        c.grad_norm_scattered([t], torch.zeros(2))
    with pytest.raises(ValueError, match="CUDA"):
        c.fused_adamw_scattered([t], [t], t, t, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0)
    with pytest.raises(ValueError, match="no weights"):
        c.fused_adamw_scattered(coco.TensorList([t], None), None, t, t, 1e-3, 0.9, 0.999, 1e-8, 0.0, 0)
    with pytest.raises(ValueError, match="copy"):
        coco.TensorList([t], [t], lps=[t.half(), t.half()])
    with pytest.raises(ValueError, match="no_decay"):
        coco.TensorList([t], [t], no_decay=[True, False])


@pytest.mark.parametrize("R", [1, 2, 3, 8])
def test_quant_layout_places_every_tensor(R):
    counts = [1000, 8, 3, 0, 4096, 70001, 256, 255, 257, (1 << 19) + 5]
    S = coco.quant_slice_elems(counts, R)
    off, total = A.starts(counts, 256)
    assert S == A.slice_elems(counts, R, 256) and S % 256 == 0 and S * R >= total
    for b, c in enumerate(counts):
        o, r0, r1 = coco.quant_tensor_place(counts, R, b)
        assert o == off[b] and o % 256 == 0
        assert (r0, r1) == ((-1, -1) if c == 0 else (o // S, (o + c - 1) // S))
    with pytest.raises(coco.CocoError):
        coco.quant_tensor_place(counts, R, len(counts))


def test_quant_state_decodes_like_its_definition():
    m, r, s = coco.quant_state([300], 1, device="cpu")
    assert (m.numel(), r.numel(), tuple(s.shape)) == (512, 512, (2, 2))
    x, v = coco.quant_decode(m, r, s)
    assert not x.any() and not v.any()
    codes = torch.arange(256, dtype=torch.uint8)
    codes[0x7F] = codes[0xFF] = 0    # the two codes that are no numbers
    scale = torch.tensor([[100, 130]], dtype=torch.uint8)
    x, v = coco.quant_decode(codes, codes & 0x7F, scale)
    assert np.array_equal(x.double().numpy(), A.code_values(codes.numpy()) * 2.0 ** -27)
    assert np.array_equal(v.double().numpy(), (A.code_values(codes.numpy() & 0x7F) * 8.0) ** 2)


def test_rounding_bits_are_even():
    """Every one of the 32 bits is set in half of 2^18 places (within 5 standard deviations), for three seeds, and
    neighbouring places agree in half of theirs."""
    n = 1 << 18
    for seed, step in ((0, 0), (1, 7), (0x123456789AB, 3)):
        b = A.rounding_bits(1 << 33, n, seed, step)
        dev = 5 * 0.5 / n ** 0.5
        for k in range(32):
            one = (b >> np.uint32(k)) & 1
            assert abs(one.mean() - 0.5) < dev, (seed, k)
            assert abs((one[1:] == one[:-1]).mean() - 0.5) < dev, (seed, k)


def test_fp32_evaluation_is_within_the_bounds_of_fp64():
    r = np.random.default_rng(0)
    n = 20000
    w, m = r.normal(0, 0.02, n).astype(np.float32), r.normal(0, 3e-4, n).astype(np.float32)
    v, g = (np.exp(r.normal(0, 1, n)) * 1e-6).astype(np.float32), r.normal(0, 1e-3, n).astype(np.float32)
    for step, dec in ((0, True), (3, False), (100000, True)):
        got = A.step32(w, m, v, g, step, dec)
        args = [x.astype(np.float64) for x in (w, m, v, g)]
        ref, err = A.step64(*args, step, dec), A.bounds64(*args, step, dec)
        for a, b, e in zip(got, ref, err):
            assert (np.abs(a - b) <= e).all()
            assert np.abs(a - b).max() > 0   # the comparison is between different computations


def test_quant_codes_round_both_ways_and_never_lose_a_positive_root():
    r = np.random.default_rng(1)
    x = (np.exp(r.normal(0, 3, 4096)) * 1e-3).astype(np.float32)
    bits = r.integers(0, 1 << 16, x.size).astype(np.uint32)
    codes, scale = A.encode32(x, bits)
    s = A.scale_values(scale).repeat(256)
    y = A.code_values(codes) * s
    step = np.exp2(np.maximum(np.floor(np.log2(np.maximum(x / s, 2.0 ** -6))), -6) - 3) * s
    assert (np.abs(y - x) <= step * (1 + 2.0 ** -20)).all() and (y > x).any() and (y < x).any()
    assert (codes < 0x79).all()          # below 448 whatever the bits
    w, m = np.zeros(512, np.float32), np.zeros(512, np.uint8)
    g = np.full(512, 1e-12, np.float32)
    g[0] = 1.0                           # the block's scale leaves the others far below the smallest code
    out = A.quant_step32(w, m, m, np.zeros((2, 2), np.uint8), g, 0, 5, 0)
    assert (out[2] > 0).all()
