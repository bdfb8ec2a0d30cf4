"""What the microscaled operators, the RMS norm and the rotary positions refuse, and the reference the GPU tests compare with.  The shape,
type and stride checks come before anything touches a device, so they run here on CPU tensors."""
import os
import re

import pytest
import torch

import mx_ref
from crowdsam_amd import hip


def mx(rows, K, fmt):
    return hip._mx_empty(torch.empty(0), rows, K, fmt)


def test_reference_formats():
    assert float(mx_ref.FP8[-1]) == 448.0 and float(mx_ref.FP8[1]) == 2.0 ** -9
    assert torch.equal(mx_ref.FP8, torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double())


def test_reference_rounds_ties_to_even_and_saturates():
    x = torch.zeros(1, 32)
    x[0, :12] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.9, -7.9, -0.25, 0.2500001])   # amax 7.9: scale 2^0
    c, s = mx_ref.quantize(x, "fp4")
    v = mx_ref.values(hip.MxTensor(c, s, "fp4", 32))
    assert int(s[0, 0, 0]) == 127
    assert v[0, :12].tolist() == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0, 6.0, -6.0, 0.0, 0.5]


@pytest.mark.parametrize("call,match", [
    (lambda: hip.mx_quantize(torch.zeros(4, 32), "fp6"), "fp6"),
    (lambda: hip.mx_quantize(torch.zeros(4, 32, dtype=torch.float64)), "float64"),
    (lambda: hip.mx_quantize(torch.zeros(4, 0)), "no columns"),
    (lambda: hip.mx_quantize(torch.zeros(32)), "dimensions"),
    (lambda: hip.mx_quantize(torch.zeros(32, 4).t()), "not contiguous"),
    (lambda: hip.mx_quantize(torch.empty(1, (1 << 31) - 100, dtype=torch.float16, device="meta")), "columns"),
    (lambda: hip.mx_quantize(torch.zeros(1, 32).expand(4, 32)), "overlap"),
    (lambda: hip.mx_quantize(torch.zeros(4, 32)), "no CPU form"),
    (lambda: hip.mx_dequantize(mx(4, 100, "fp4"), torch.int32), "int32"),
    (lambda: hip.mx_dequantize(hip.MxTensor(torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(2, 4, 4, dtype=torch.uint8), "fp4", 100)),
     "codes of shape"),
    (lambda: hip.mx_dequantize(hip.MxTensor(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(4, 2, 4, dtype=torch.uint8), "fp4", 100)),
     "scales of shape"),
    (lambda: hip.mx_dequantize(hip.MxTensor(torch.zeros(4, 136, dtype=torch.uint8)[:, 4:132], torch.zeros(2, 4, 4, dtype=torch.uint8), "fp4", 100)),
     "16-byte"),
    (lambda: hip.mx_dequantize(hip.MxTensor(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(2, 4, 8, dtype=torch.uint8)[..., ::2], "fp4", 100)),
     "4 bytes apart"),
    (lambda: hip.mx_gemm(mx(4, 256, "fp8"), mx(8, 256, "fp8")), "only 'fp4' weights"),
    (lambda: hip.mx_gemm(mx(4, 256, "fp8"), mx(8, 250, "fp4")), "K = 256"),
    (lambda: hip.mx_gemm(mx(4, 256, "fp8"), mx(8, 256, "fp4"), bias=torch.zeros(4)), "bias"),
    (lambda: hip.mx_gemm(mx(4, 256, "fp8"), mx(8, 256, "fp4"), bias=torch.zeros(8, dtype=torch.float16)), "bias"),
    (lambda: hip.mx_gemm(mx(4, 256, "fp8"), mx(8, 256, "fp4"), residual=torch.zeros(8, 4)), "residual"),
    (lambda: hip.mx_gemm(mx(4, 256, "fp8"), mx(8, 256, "fp4"), out=torch.zeros(4, 9)), "out has shape"),
    (lambda: hip.mx_gemm(mx(4, 256, "fp8"), mx(8, 256, "fp4"), act=7), "activation"),
    (lambda: hip.mx_gemm(hip.MxTensor(torch.empty(2, 1 << 24, dtype=torch.uint8)[:, :256], *mx(2, 256, "fp8")[1:]), mx(8, 256, "fp4")), "2\\^24"),
    (lambda: hip.mx_gemm(mx(4, 256, "fp8"), mx(8, 256, "fp4"), out_dtype=torch.float64), "float64"),
    (lambda: hip.mx_gemm(mx(4, 256, "fp8"), mx(8, 256, "fp4")), "no CPU form"),
    (lambda: hip.rms_norm(torch.zeros(4, 64), torch.zeros(64), 0.0), "eps"),
    (lambda: hip.rms_norm(torch.zeros(4, 64), torch.zeros(64), float("nan")), "eps"),
    (lambda: hip.rms_norm(torch.zeros(4, 64), torch.zeros(63), 1e-6), "gamma"),
    (lambda: hip.rms_norm(torch.zeros(4, 64), torch.zeros(64, dtype=torch.float16), 1e-6), "gamma"),
    (lambda: hip.rms_norm(torch.zeros(1, 32769), torch.zeros(32769), 1e-6), "32768"),
    (lambda: hip.rms_norm(torch.zeros(4, 64), torch.zeros(64), 1e-6, residual=torch.zeros(4, 64, dtype=torch.float16)), "residual"),
    (lambda: hip.rms_norm(torch.zeros(4, 64), torch.zeros(64), 1e-6, residual=torch.zeros(3, 64)), "residual"),
    (lambda: hip.rms_norm(torch.zeros(4, 64), torch.zeros(64), 1e-6, h_out=torch.zeros(4, 64)), "without a residual"),
    (lambda: hip.rms_norm(torch.zeros(4, 64), torch.zeros(64), 1e-6, residual=torch.zeros(4, 64), h_out=torch.zeros(4, 64).half()), "h_out"),
    (lambda: hip.rms_norm(torch.zeros(4, 64), torch.zeros(64), 1e-6, out_dtype="fp6"), "fp6"),
    (lambda: hip.rms_norm(torch.zeros(4, 64), torch.zeros(64), 1e-6), "no CPU form"),
])
def test_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def rot(q=None, k=None, pos=None, pairs=8, axes=2, **kw):
    q = torch.zeros(6, 2, 32) if q is None else q
    pos = torch.zeros(axes, 6) if pos is None else pos
    freq, axis = hip.rotary_frequencies([pairs // 2, pairs - pairs // 2], device="cpu")
    return hip.rotary(q, k, pos, kw.pop("freq", freq), kw.pop("axis", axis), **kw)


@pytest.mark.parametrize("call,match", [
    (lambda: rot(q=torch.zeros(6, 64)), "dimensions"),
    (lambda: rot(q=torch.zeros(6, 2, 32, dtype=torch.float64)), "float64"),
    (lambda: rot(pairs=17), "17 pairs"),
    (lambda: rot(q=torch.zeros(6, 1, 4098)), "4096"),
    (lambda: rot(pos=torch.zeros(2, 4)), "multiple"),
    (lambda: rot(pos=torch.zeros(2, 6, dtype=torch.int64)), "pos"),
    (lambda: rot(pos=torch.zeros(6, 2).t()), "positions of an axis"),
    (lambda: rot(freq=torch.zeros(8)), "float64"),
    (lambda: rot(axis=torch.zeros(8, dtype=torch.int64)), "int32"),
    (lambda: rot(k=torch.zeros(5, 2, 32)), "k has shape"),
    (lambda: rot(k=torch.zeros(6, 2, 32, dtype=torch.float16)), "float16"),
    (lambda: rot(k_out=torch.zeros(6, 2, 32)), "without k"),
    (lambda: rot(q_out=torch.zeros(6, 3, 32)), "q_out has shape"),
    (lambda: rot(q_out=torch.zeros(1, 2, 32).expand(6, 2, 32)), "overlap"),
    (lambda: rot(q=torch.zeros(6, 32, 2).transpose(1, 2)), "not contiguous"),
    (lambda: rot(), "no CPU form"),
    (lambda: hip.rotary_frequencies([4, 0]), "sections"),
])
def test_rotary_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()


def test_entries_check_for_themselves():
    """The C entries refuse what the wrappers would have caught (no device is touched)."""
    lib = hip.lib()
    assert lib.csam_mx_quantize(None, None, 0, 0, None, 0, None, 0, 0, 1, 1) == -1 and b"null" in lib.csam_last_error()
    assert lib.csam_mx_quantize(None, 64, 32, 0, 64, 128, 64, 4, 2, 1, 32) == -1 and b"format" in lib.csam_last_error()
    assert lib.csam_mx_quantize(None, 64, 32, 0, 64, 120, 64, 4, 0, 1, 32) == -1 and b"padded" in lib.csam_last_error()
    assert lib.csam_mx_quantize(None, 64, 1, 0, 64, 128, 64, 1 << 33, 0, (1 << 31) - 1, 1) == -1 and b"2^31" in lib.csam_last_error()
    assert lib.csam_mx_gemm(None, 64, 128, 64, 1 << 33, 0, 64, 128, 64, 4, 64, 1, 0, None, None, 0, 0, 0, (1 << 31) - 1, 1, 32) == -1 and \
        b"2^31" in lib.csam_last_error()
    assert lib.csam_mx_dequantize(None, 64, 128, 64, 4, 0, 64, 31, 0, 1, 32) == -1 and b"sizes" in lib.csam_last_error()
    assert lib.csam_mx_gemm(None, 64, 128, 64, 4, 0, 72, 128, 64, 4, 64, 1, 0, None, None, 0, 0, 0, 1, 1, 32) == -1 and b"16 bytes" in lib.csam_last_error()
    assert lib.csam_rms_norm(None, 64, 8, 0, 64, 8, 0, None, 8, 64, 1e-6, 64, 8, 0, 1, 8) == -1 and b"together" in lib.csam_last_error()
    assert lib.csam_rotary(None, 64, 8, 8, 64, 8, 8, 1, None, 0, 0, None, 0, 0, 0, 0, 64, 1, 0, 64, 64, 1, 5, 0, 1, 1, 8) == -1 and \
        b"pairs" in lib.csam_last_error()


def test_gelu_polynomial_is_within_its_bound():
    """The polynomial of Phi that 16-bit results take (csrc/csam_common.h), in float64 over the reals: |x P(x) - x Phi(x)| < 6.5e-5.  Beyond
    the clamp both sides are within x (1 - Phi(x)) of each other, which only falls there."""
    src = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "crowdsam_amd", "csrc", "csam_common.h")).read()
    body = src[src.index("csam_gelu_poly2(float2_t x)"):]
    c = float(re.search(r"const float c = ([0-9.]+)f;", body)[1])
    k = [float(v) for v in re.search(r"k\[9\] = \{(.*?)\};", body, re.S)[1].replace("f", "").split(",")]
    x = torch.linspace(-12, 12, 2_400_001, dtype=torch.float64)
    xc = x.clamp(-c, c)
    r = torch.full_like(x, k[0])
    for v in k[1:]:
        r = r * xc * xc + v
    off = (x * (0.5 + xc * r) - x * 0.5 * torch.special.erfc(-x / 2 ** 0.5)).abs()
    assert len(k) == 9 and float(off.max()) < 6.5e-5
