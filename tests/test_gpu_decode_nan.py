"""Decode over keys whose scores are NaN, or -inf, a whole run of them: chunks and quarters of a sequence without one
finite score. A row that sees a NaN is NaN wherever the NaN lies; keys at -inf have weight 0."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
DT = {"fp16": torch.float16, "bf16": torch.bfloat16}
N, PAGE, HKV = 1600, 16, 2
BLOCKS = N // 16


def runs():
    """Runs of whole blocks [a, b): from the front, up to the end, and inside (the sequence's chunks and the merge's quarters
    of them end somewhere among these)."""
    out = [(0, b) for b in range(1, BLOCKS, 3)] + [(a, BLOCKS) for a in range(1, BLOCKS, 3)]
    return out + [(a, a + n) for n in (13, 25, 26, 50) for a in range(1, BLOCKS - n, 6)]


def i32(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device=DEV)


def table():
    return i32([0, BLOCKS]), i32(range(1, BLOCKS + 1)), i32([16])


@pytest.mark.parametrize("code", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype,d", [("fp16", 64), ("bf16", 128), ("fp16", 256)])
def test_8_bit_decode_of_runs_that_are_not_finite(dtype, d, code):
    from nanoslg_amd import kernels as K
    g = torch.Generator(device=DEV).manual_seed(1)
    k = torch.randint(-60, 61, (BLOCKS + 1, PAGE, HKV, d), generator=g, device=DEV)
    k, v = ((x if code == "int8" else x.float()).to(torch.int8 if code == "int8" else torch.float8_e4m3fn) for x in (k, k.flip(0)))
    ks, vs = (torch.full((BLOCKS + 1, 1, HKV), 2.0 ** -6, device=DEV) for _ in "kv")
    q = torch.randn(1, 4 * HKV, d, generator=g, device=DEV).to(DT[dtype])
    want = K.paged_decode_q8(q, k, v, ks, vs, *table(), BLOCKS)
    assert torch.isfinite(want).all()
    for a, b in runs():
        k2, ks2 = k.clone(), ks.clone()
        if code == "int8":
            ks2[1 + a:1 + b, :, 0] = math.nan
        else:
            k2.view(torch.int8)[1 + a:1 + b, :, 0] = 0x7f
        out = K.paged_decode_q8(q, k2, v, ks2, vs, *table(), BLOCKS)
        assert torch.isnan(out[0, :4]).all(), (a, b)
        assert torch.equal(out[0, 4:], want[0, 4:]), (a, b)


@pytest.mark.parametrize("dtype,d", [("fp16", 64), ("bf16", 128), ("fp16", 256)])
def test_16_bit_decode_of_runs_that_are_not_finite(dtype, d):
    from nanoslg_amd import kernels as K
    g = torch.Generator(device=DEV).manual_seed(2)
    k, v = (torch.randn(BLOCKS + 1, PAGE, HKV, d, generator=g, device=DEV).to(DT[dtype]) for _ in "kv")
    q = torch.randn(1, 4 * HKV, d, generator=g, device=DEV).to(DT[dtype])
    want = K.paged_decode(q, k, v, *table(), BLOCKS)
    for a, b in runs():
        k2 = k.clone()
        k2[1 + a:1 + b, :, 0] = math.nan
        out = K.paged_decode(q, k2, v, *table(), BLOCKS)
        assert torch.isnan(out[0, :4]).all(), (a, b)
        assert torch.equal(out[0, 4:], want[0, 4:]), (a, b)


@pytest.mark.parametrize("dtype,d", [("fp16", 64), ("bf16", 128), ("fp16", 256)])
def test_16_bit_decode_of_runs_at_minus_infinity(dtype, d):
    """One channel of K at -inf where q has a positive value and zeros everywhere else: those keys have weight 0, and the
    row is the mean of the other keys' V."""
    from nanoslg_amd import kernels as K
    g = torch.Generator(device=DEV).manual_seed(3)
    k = torch.zeros(BLOCKS + 1, PAGE, HKV, d, device=DEV, dtype=DT[dtype])
    v = torch.randint(-8, 9, (BLOCKS + 1, PAGE, HKV, d), generator=g, device=DEV).to(DT[dtype])
    q = torch.ones(1, 4 * HKV, d, device=DEV, dtype=DT[dtype])
    for a, b in runs():
        k2 = k.clone()
        k2[1 + a:1 + b, :, 0, 5] = -math.inf
        out = K.paged_decode(q, k2, v, *table(), BLOCKS)[0, :4].double()
        keep = torch.cat([v[1:1 + a, :, 0], v[1 + b:, :, 0]]).reshape(-1, d).double()
        want = keep.mean(0).expand(4, d)
        # weights are exactly 1 (or one power of two), V's sums whole numbers below 2^24: the quotient (by a reciprocal and
        # a product, 2^-22 in all) and the output's rounding remain
        step = 2.0 ** -11 if dtype == "fp16" else 2.0 ** -8
        assert ((out - want).abs() <= want.abs() * (step + 2.0 ** -21) + 2.0 ** -24).all(), (a, b)
