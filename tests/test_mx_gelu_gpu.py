"""GELU of hip.mx_gemm where a polynomial goes wrong: far negative and far positive values, next to zero, the ends of the range."""
import pytest
import torch

from test_mx_gpu import U, close, gen, operands, product_ref

pytestmark = pytest.mark.gpu


def values(n):
    """n pre-activations: -6.5 .. 6.5, the far ends, powers of two next to zero."""
    far = torch.tensor([7.0, 8.5, 10.0, 50.0, 100.0, 1000.0, 10000.0])
    small = torch.exp2(-torch.arange(1.0, 14.0))
    x = torch.cat((far, -far, small, -small, torch.zeros(1)))
    return torch.cat((x, torch.linspace(-6.5, 6.5, n - len(x))))


# one row and few rows (the direct form), 64-wide, 128-wide tiles and past them 256-wide ones
@pytest.mark.parametrize("fa", ["fp4", "fp8"])
@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n", [(1, 4096), (20, 130), (300, 513), (2100, 2003), (4000, 4090)])
def test_gelu_of_every_size(cuda, fa, out_dtype, m, n):
    """Zero rows and a bias: the activation's argument is the bias itself, so the only errors are the activation's own and the store's.
    16 bits: 6e-6 of the result up to 6.25 (test_mx_gelu_cpu; the exponential is off by an ulp more, 2 U) and 1.3e-9 beyond.
    fp32: x (1 + e) / 2 with e = 1 - p(t) t exp(-z^2), z = |x| / sqrt 2, t = 1 / (1 + 0.33 z), off by 1.5e-7 as a formula.  Its roundings:
    z, times e'(z) z <= 0.49, with the constant's 1 U; t by 3 U at most (the sum, the reciprocal to an ulp), times |(p t)'| t exp(-z^2), whose
    largest value is 1 at t = 0.75 .. 1, where t itself is exact at 1: 3 U; Horner's four sums, of values below 1.45, 1.43, 1.14 and 1 while t
    <= 1: 5 U; the exponential, its argument's two roundings times z^2 exp(-z^2) <= 0.37 and an ulp: 3 U; two products of values below 1:
    2 U; the difference and 1 + e: 2 U.  Together 16 U in e, half of it times |x|, and the last product.  Beyond 6 the part taken from 1 is
    below 1e-8, less than half a step of 1: e is 1."""
    from crowdsam_amd import hip
    bias = values(n)
    qa, qw = hip.mx_quantize(torch.zeros(m, 64, device=cuda), fa), hip.mx_quantize(torch.randn(n, 64, generator=gen(1)).to(cuda), "fp4")
    out = hip.mx_gemm(qa, qw, bias=bias.to(cuda), act=hip.ACT_GELU, out_dtype=out_dtype).cpu()
    x = bias.double()
    ref = x * 0.5 * torch.special.erfc(-x / 2 ** 0.5)
    f = torch.finfo(out_dtype)
    if out_dtype == torch.float32:
        own = (0.75e-7 + 8 * U) * x.abs() * (x.abs() <= 6.0) + U * ref.abs() + (x < -6.0) * ref.abs()
    else:
        own = (6e-6 + 2 * U) * ref.abs() + 1.3e-9
    close(out, ref.expand(m, n), ((own + f.eps / 2 * ref.abs() + f.smallest_normal * f.eps) * (1 + 2.0 ** -7)).expand(m, n))


@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [2, 500])
def test_gelu_at_the_ends(cuda, out_dtype, m):
    """As x (1 + erf) / 2 gives them: inf, NaN for -inf, NaN."""
    from crowdsam_amd import hip
    bias = torch.zeros(300)
    bias[0], bias[1], bias[2] = float("inf"), float("-inf"), float("nan")
    qa, qw = hip.mx_quantize(torch.zeros(m, 64, device=cuda), "fp8"), hip.mx_quantize(torch.ones(300, 64, device=cuda), "fp4")
    out = hip.mx_gemm(qa, qw, bias=bias.to(cuda), act=hip.ACT_GELU, out_dtype=out_dtype).cpu().float()
    assert bool((out[:, 0] == float("inf")).all()) and bool(out[:, 1:3].isnan().all()) and bool((out[:, 3:] == 0).all())


@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m", [1, 100, 2100])
def test_gelu_of_a_product(cuda, out_dtype, m):
    """E2M1 products (whose sums lose nothing) through GELU: nothing but the sum's fp32 error, 6e-6 of the result and the store's rounding."""
    from crowdsam_amd import hip
    n, k = 2050, 300
    a, w = operands(m, n, k, "fp4", 31 + m)
    bias = torch.randn(n, generator=gen(5)) * 3 - 3
    qa, qw = hip.mx_quantize(a.to(cuda), "fp4"), hip.mx_quantize(w.to(cuda), "fp4")
    x, tol = product_ref(hip, qa, qw, bias, 0, None, torch.float32)
    ref = x * 0.5 * torch.special.erfc(-x / 2 ** 0.5)
    f = torch.finfo(out_dtype)
    tol = 1.13 * tol + 6e-6 * ref.abs() + 1.3e-9 + f.eps / 2 * ref.abs() + f.smallest_normal * f.eps
    close(hip.mx_gemm(qa, qw, bias=bias.to(cuda), act=hip.ACT_GELU, out_dtype=out_dtype), ref, tol * (1 + 2.0 ** -7))
