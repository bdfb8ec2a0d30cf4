"""hip.rms_norm against float64."""
import pytest
import torch

import mx_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
EPS = 1e-6


def rows(m, d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, d, generator=g) + torch.randn(d, generator=g) * 0.3
    x[:, d // 2] += 40.0
    return x.to(dtype)


def check(out, ref, dtype, fp32_steps):
    tol = ref.abs() * (fp32_steps * U + torch.finfo(dtype).eps / 2) * (1 + 2.0 ** -7) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    d = (out.cpu().double() - ref).abs()
    assert bool((d <= tol).all()), float((d / tol).max())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("res", [None, "same", torch.float32])
@pytest.mark.parametrize("m,d", [(1, 1), (1, 8), (5, 31), (2, 512), (7, 520), (9, 1024), (3, 1280), (4, 2048), (6, 2056), (1, 2047), (3, 8192),
                                 (2, 8200), (1, 32768), (40, 1001)])
def test_matches_float64(cuda, dtype, res, m, d):
    """Squares and their sum: a lane adds up to 32 of them in turn, then 6 levels of lanes and up to 16 waves: 54 roundings of positive
    terms, half of that after the root; h, the mean, eps, the root, the quotient and the two factors: 7 more; 40 steps cover it."""
    from crowdsam_amd import hip
    x = rows(m, d, dtype, m + d)
    gamma = torch.rand(d, generator=torch.Generator().manual_seed(1)) + 0.5
    r = None if res is None else rows(m, d, dtype if res == "same" else res, m * d + 1)
    h = x.double() if r is None else x.double() + r.double()
    ref = h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS) * gamma.double()
    xs, gs = x.to(cuda), gamma.to(cuda)
    f32 = None
    for out_dtype in (torch.float32, torch.float16, torch.bfloat16, "fp8", "fp4"):
        if r is None:
            y = hip.rms_norm(xs, gs, EPS, out_dtype=out_dtype)
        else:
            rs = r.to(cuda)
            y, ho = hip.rms_norm(xs, gs, EPS, residual=rs, out_dtype=out_dtype)
            assert torch.equal(rs.cpu(), r)
            check(ho, h, r.dtype, 1)
            y2, h2 = hip.rms_norm(xs, gs, EPS, residual=rs, h_out=rs, out_dtype=out_dtype)        # in place
            assert h2.data_ptr() == rs.data_ptr() and torch.equal(h2, ho)
        if out_dtype in ("fp8", "fp4"):                     # the same row, then the definition of the format
            codes, scales = mx_ref.quantize(f32, out_dtype)
            assert y.K == d and torch.equal(y.codes.cpu(), codes) and torch.equal(y.scales.cpu(), scales)
        else:
            check(y, ref, out_dtype, 40)
            f32 = y.cpu() if out_dtype == torch.float32 else f32


def test_strides(cuda):
    from crowdsam_amd import hip
    base = rows(50, 700, torch.float16, 3)
    gamma = torch.rand(320, generator=torch.Generator().manual_seed(1)) + 0.5
    for off in (0, 8, 5):
        x, r = base[:, off:off + 320], base[:, 360 + off % 8:680 + off % 8]
        h = x.double() + r.double()
        ref = h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS) * gamma.double()
        d = base.to(cuda)
        y, ho = hip.rms_norm(d[:, off:off + 320], gamma.to(cuda), EPS, residual=d[:, 360 + off % 8:680 + off % 8], out_dtype=torch.float32)
        check(y, ref, torch.float32, 40)
        check(ho, h, torch.float16, 1)


def test_many_rows_and_zero_rows(cuda):
    """More rows than a launch has workgroups for at one row each; a row of zeros stays zero; a row with a NaN is NaN alone."""
    from crowdsam_amd import hip
    x = rows(20011, 256, torch.bfloat16, 2)
    x[17] = 0
    x[20010, 3] = float("nan")
    gamma = torch.ones(256)
    y = hip.rms_norm(x.to(cuda), gamma.to(cuda), EPS, out_dtype=torch.float32).cpu()
    h = x.double()
    ref = h / torch.sqrt(h.square().mean(1, keepdim=True) + EPS)
    check(y[:20010], ref[:20010], torch.float32, 40)
    assert bool((y[17] == 0).all()) and bool(torch.isnan(y[20010]).all())
    q = hip.rms_norm(x.to(cuda), gamma.to(cuda), EPS, out_dtype="fp4")
    codes, scales = mx_ref.quantize(y, "fp4")
    assert torch.equal(q.codes.cpu(), codes) and torch.equal(q.scales.cpu(), scales)
