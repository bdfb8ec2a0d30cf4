"""The GELU of 16-bit products (csrc/mx_gemm.hip), evaluated here as the kernel does: fp32, fused multiply-adds, over the whole line."""
import os
import re

import numpy as np
import torch

F = np.float32


def coefficients():
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "crowdsam_amd", "csrc", "mx_gemm.hip")).read()
    body = src[src.index("float mx_gelu16(float x)"):]
    return [F(v) for v in re.search(r"k\[8\] = \{(.*?)\};", body, re.S)[1].replace("f", "").split(",")]


def gelu(x):
    """x as float32; a product of two fp32 numbers is exact in float64, so the sum rounds once but for a double rounding in 2^29."""
    a, k = np.abs(x), coefficients()
    assert len(k) == 8
    r = np.full_like(a, k[0])
    for v in k[1:]:
        r = (r.astype(np.float64) * a.astype(np.float64) + np.float64(v)).astype(F)
    q = np.exp2(r.astype(np.float64)).astype(F)
    return x * np.where(x < 0, q, F(1) - q)


def exact(x):
    x = torch.from_numpy(x.astype(np.float64))
    return (x * 0.5 * torch.special.erfc(-x / 2 ** 0.5)).numpy()


def test_gelu_is_within_its_bound_everywhere():
    """6e-6 of the result up to |x| = 6.25 and 1.3e-9 beyond: under a hundredth of half an fp16 step, and no term that grows with |x|."""
    x = np.concatenate((np.linspace(-13, 13, 2_600_001), np.geomspace(1e-30, 1e-3, 1000), -np.geomspace(1e-30, 1e-3, 1000))).astype(F)
    off, ref = np.abs(gelu(x).astype(np.float64) - exact(x)), np.abs(exact(x))
    near = np.abs(x) <= 6.25
    assert bool((off <= 6e-6 * ref)[near].all())
    assert float(off[x < -6.25].max()) <= 1.3e-9 and bool((off <= 1e-8 * ref)[x > 6.25].all())


def test_gelu_far_away_and_not_finite():
    with np.errstate(all="ignore"):
        far = np.array([13, 50, 100, 1e4, 65504, 1e20, 3e38], F)
        assert bool((gelu(far) == far).all()) and bool((np.abs(gelu(-far)) <= 1e-37).all())
        ends = gelu(np.array([np.inf, -np.inf, np.nan, 0.0], F))
    # as x (1 + erf) / 2 gives them
    assert ends[0] == np.inf and np.isnan(ends[1]) and np.isnan(ends[2]) and ends[3] == 0


def test_stated_bounds_of_the_packed_polynomial():
    """csam_common.h states of csam_gelu_poly2, the detector's GELU: 4.1e-5 below 3, 8.1e-5 up to the clamp, 1.4e-6 |x| beyond.  Every fp32
    value about the largest error, in the order that the kernel evaluates."""
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "crowdsam_amd", "csrc", "csam_common.h")).read()
    body = src[src.index("csam_gelu_poly2(float2_t x)"):]
    c = F(re.search(r"const float c = ([0-9.]+)f;", body)[1])
    k = [F(v) for v in re.search(r"k\[9\] = \{(.*?)\};", body, re.S)[1].replace("f", "").split(",")]

    def fma(a, b, d):
        return (a.astype(np.float64) * b.astype(np.float64) + np.float64(d)).astype(F)

    def off(x):
        xc = np.clip(x, -c, c)
        u, r = xc * xc, np.full_like(x, k[0])
        for v in k[1:]:
            r = fma(r, u, v)
        return np.abs((x * fma(xc, r, F(0.5))).astype(np.float64) - exact(x))

    about = np.arange(F(4.2).view(np.int32), F(4.4).view(np.int32), dtype=np.int32).view(F)
    x = np.concatenate((np.linspace(-4.4, 4.4, 880_001).astype(F), about, -about))
    e = off(x)
    assert 8.0e-5 < float(e.max()) <= 8.1e-5 and float(e[np.abs(x) < 3].max()) <= 4.1e-5
    far = np.geomspace(4.4, 6e4, 2001).astype(F)
    assert bool((off(far) <= 8.1e-5 + 1.4e-6 * far).all()) and bool((off(-far) <= 8.1e-5 + 1.4e-6 * far).all())
    assert bool((off(-far[far > 20]) <= 1.4e-6 * far[far > 20]).all())
