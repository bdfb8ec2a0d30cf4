"""hip.mx_gemm of an E4M3 operand where the scaled matrix instruction drops bits: sums that fp32 holds exactly in any order and that need
bits far below 2^-13 of a neighbouring product."""
import pytest
import torch

import mx_ref
from test_mx_gpu import gen

pytestmark = pytest.mark.gpu


def fine(m, n, k, seed):
    """(qa, qw, float64 product).  Of 16 neighbours of a row of A one is +-256, the others are multiples of 2^-9 below 2^-3; W holds +-1/2 and
    +-1.  Every product is a multiple of 2^-10 and every sum of k <= 512 is below 32 x 256 + 512 / 8 < 2^14: 24 bits, exact in any order.
    The matrix instruction keeps 2^-5 of a group that 256 leads."""
    from crowdsam_amd import hip
    g = gen(seed)
    small = torch.cat((torch.arange(8.0) * 2.0 ** -9, (8 + torch.arange(8.0)) * 2.0 ** -8, (8 + torch.arange(8.0)) * 2.0 ** -7))
    a = small[torch.randint(0, len(small), (m, k), generator=g)]
    at = torch.randint(0, 16, (m, -(-k // 16)), generator=g) + 16 * torch.arange(-(-k // 16))
    a.scatter_(1, at.clamp(max=k - 1), 256.0)
    a = a * (torch.randint(0, 2, (m, k), generator=g) * 2 - 1)
    w = torch.tensor([0.5, -0.5, 1.0, -1.0])[torch.randint(0, 4, (n, k), generator=g)]
    w[:, ::32] = 1.0
    qa, qw = hip.mx_quantize(a.cuda(), "fp8"), hip.mx_quantize(w.cuda(), "fp4")
    assert torch.equal(mx_ref.values(qa), a.double()) and torch.equal(mx_ref.values(qw), w.double())
    return qa, qw, a.double() @ w.double().t()


def scaled(q, powers, rows=None):
    """``q`` with the scale bytes of its blocks moved by ``powers`` [groups of 128 columns], of all rows or those given (blocks behind K
    stay)."""
    groups, m, _ = q.scales.shape
    by = torch.as_tensor(powers, dtype=torch.int32).view(-1, 1, 1).expand(groups, m, 4).clone()
    by[(torch.arange(groups * 4) >= -(-q.K // 32)).view(groups, 1, 4).expand_as(by)] = 0
    if rows is not None:
        keep = torch.ones(m, dtype=torch.bool)
        keep[rows] = False
        by[:, keep] = 0
    s = q.scales.int() + by.to(q.scales.device)
    assert 0 <= int(s.min()) and int(s.max()) < 255
    return q._replace(scales=s.to(torch.uint8))


# one row and few rows (the direct form with one and with two tiles of 16 rows); 64-wide tiles; 128-wide tiles, whole and ragged
SHAPES = [(1, 64, 256), (3, 130, 512), (16, 260, 500), (33, 40, 256), (200, 300, 512), (511, 130, 300), (2048, 2048, 256), (2100, 2001, 300),
          (1, 4096, 512), (7, 1, 32), (100, 1000, 300), (300, 900, 300)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_fp32_results_lose_nothing(cuda, m, n, k):
    from crowdsam_amd import hip
    qa, qw, ref = fine(m, n, k, m + n)
    assert torch.equal(hip.mx_gemm(qa, qw, out_dtype=torch.float32).cpu().double(), ref)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_fp32_results_lose_nothing_at_any_scale(cuda, m, n, k):
    """The same values with their scales moved to the ends of the range, undone in the other operand: the same bits."""
    from crowdsam_amd import hip
    qa, qw, ref = fine(m, n, k, m + n + 1)
    groups = qa.scales.shape[0]
    by = torch.tensor([0, 125, -120, 97])[torch.arange(groups) % 4]
    out = hip.mx_gemm(scaled(qa, by), scaled(qw, -by), out_dtype=torch.float32)
    assert torch.equal(out.cpu().double(), ref)


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_rows_at_the_ends_of_the_range_leave_the_others_whole(cuda, m, n, k):
    """Rows of A and of W with far scales of their own: their results are moved by the same power of two, the others keep every bit.  A row
    that is too small for fp32 becomes what fp32 makes of it; a NaN block is its row's alone."""
    from crowdsam_amd import hip
    qa, qw, ref = fine(m, n, k, m + n + 2)
    groups = qa.scales.shape[0]
    up, down = m // 2, m - 1
    qa = scaled(qa, [100] * groups, [up])
    if down != up:
        qa = scaled(qa, [-100] * groups, [down])
    qw = scaled(qw, [-110] * groups, [n // 2])
    power = torch.zeros(m, n, dtype=torch.float64)
    power[up] += 100
    if down != up:
        power[down] -= 100
    power[:, n // 2] -= 110
    want = (ref * torch.exp2(power)).float()
    out = hip.mx_gemm(qa, qw, out_dtype=torch.float32).cpu()
    tiny = want.abs() < 2.0 ** -126                        # (fp32 may flush them)
    assert torch.equal(out[~tiny], want[~tiny]) and float(out[tiny].abs().max() if tiny.any() else 0) < 2.0 ** -125
    s = qw.scales.clone()
    s[1, 0, 2] = 255
    out = hip.mx_gemm(qa, qw._replace(scales=s), out_dtype=torch.float32).cpu()
    assert bool(out[:, 0].isnan().all()) and torch.equal(out[:, 1:][~tiny[:, 1:]], want[:, 1:][~tiny[:, 1:]])


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_the_cut_stays_in_its_bound_and_shows(cuda, m, n, k):
    """``cut``: each of the 15 neighbours of a group loses less than 2^-13 of the group's largest product, 2^-5 here, in ceil(k / 16) groups.
    Many rows show it, so the tests above can tell the two apart."""
    from crowdsam_amd import hip
    qa, qw, ref = fine(m, n, k, m + n)
    d = (hip.mx_gemm(qa, qw, out_dtype=torch.float32, cut=True).cpu().double() - ref).abs()
    assert float(d.max()) <= 15 * 2.0 ** -5 * -(-k // 16)
    if m >= 200:
        assert float(d.max()) > 0


@pytest.mark.parametrize("out_dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_16_bit_results_lose_nothing_if_asked(cuda, out_dtype, m, n, k):
    """cut=False: the exact sum, rounded once.  With no choice made that holds for few rows; many rows stay in the cut's bound."""
    from crowdsam_amd import hip
    qa, qw, ref = fine(m, n, k, m + n)
    want = ref.to(out_dtype)                               # (ref is an fp32 value: one rounding)
    assert torch.equal(hip.mx_gemm(qa, qw, out_dtype=out_dtype, cut=False).cpu(), want)
    out = hip.mx_gemm(qa, qw, out_dtype=out_dtype).cpu()
    if m <= 16 or -(-m // 16) * -(-n // 16) <= 512:
        assert torch.equal(out, want)
    else:
        lost = 15 * 2.0 ** -5 * -(-k // 16)
        assert float((out.double() - ref).abs().max()) <= lost + torch.finfo(out_dtype).eps / 2 * (float(ref.abs().max()) + lost)


@pytest.mark.parametrize("m", [5, 300, 2100])
def test_the_choice_with_an_epilogue(cuda, m):
    """Bias, activation and residual behind a sum that lost nothing: integers of 1/4 that fp32 and fp16 hold, so the result is exact."""
    from crowdsam_amd import hip
    n, k = 2000, 256
    g = gen(m)
    a = torch.zeros(m, k)
    a[:, 0], a[:, 1], a[:, 2] = 256.0, -256.0, 0.0625 * torch.randint(1, 16, (m,), generator=g)     # 2^-4 beside 2^8
    w = torch.ones(n, k)
    qa, qw = hip.mx_quantize(a.to(cuda), "fp8"), hip.mx_quantize(w.to(cuda), "fp4")
    assert torch.equal(mx_ref.values(qa), a.double())
    bias, res = 0.25 * torch.randint(-8, 9, (n,), generator=g), 0.25 * torch.randint(-8, 9, (m, n), generator=g)
    out = hip.mx_gemm(qa, qw, bias=bias.float().to(cuda), act=hip.ACT_RELU, residual=res.half().to(cuda), cut=False)
    ref = (a[:, 2].double()[:, None] + bias.double()).clamp(min=0) + res.double()
    assert torch.equal(out.cpu(), ref.half())


def test_the_choice_changes_nothing_for_e2m1(cuda):
    from crowdsam_amd import hip
    for m in (4, 700):
        qa = hip.mx_quantize(torch.randn(m, 300, generator=gen(m)).to(cuda), "fp4")
        qw = hip.mx_quantize(torch.randn(900, 300, generator=gen(1)).to(cuda), "fp4")
        outs = [hip.mx_gemm(qa, qw, out_dtype=torch.float32, cut=cut) for cut in (None, False, True)]
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@pytest.mark.parametrize("cut", [None, False, True])
@pytest.mark.parametrize("m,n,k", [(3, 130, 512), (100, 1000, 300), (300, 900, 300), (2100, 2001, 300)])
def test_nan_codes(cuda, m, n, k, cut):
    """E4M3's NaN code, which quantisation never writes: its row becomes NaN, the others keep what they were."""
    from crowdsam_amd import hip
    qa, qw, _ = fine(m, n, k, m + n)
    whole = hip.mx_gemm(qa, qw, out_dtype=torch.float32, cut=cut)
    codes = qa.codes.clone()
    codes[1, k // 2], codes[m - 1, 3] = 0x7F, 0xFF
    out = hip.mx_gemm(qa._replace(codes=codes), qw, out_dtype=torch.float32, cut=cut)
    bad = torch.zeros(m, dtype=torch.bool, device=cuda)
    bad[1] = bad[m - 1] = True
    assert bool(out[bad].isnan().all()) and torch.equal(out[~bad], whole[~bad])


@pytest.mark.parametrize("at", [(-59, -59), (-62, -70), (-118, 0), (0, -118)])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_products_below_the_normal_range(cuda, at, m, n, k):
    """Sums of normal size of products that are subnormal: multiples of 2^-10 times 2^-118 or 2^-132, which fp32 holds."""
    from crowdsam_amd import hip
    qa, qw, ref = fine(m, n, k, m + n + 3)
    groups = qa.scales.shape[0]
    out = hip.mx_gemm(scaled(qa, [at[0]] * groups), scaled(qw, [at[1]] * groups), out_dtype=torch.float32)
    assert torch.equal(out.cpu().double(), ref * 2.0 ** sum(at))
