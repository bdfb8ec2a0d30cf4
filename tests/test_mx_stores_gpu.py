"""Results that are stored past the caches: large products whose rows are whole lines, and quantised, dequantised, normed and rotated rows of
more bytes than the caches hold.  Each against float64, and bit for bit against the same rows in calls too small for it."""
import pytest
import torch

import mx_ref
from test_mx_gpu import U, equal, gen, group_max, operands
from test_rms_norm_gpu import EPS
from test_rotary_gpu import check as check_rotary, positions

pytestmark = pytest.mark.gpu
DTS = [torch.float16, torch.bfloat16, torch.float32]


# 128 x 128 (both step widths of E2M1), 128 x 256 and 256 x 256 tiles; E4M3 with nothing dropped; every N is whole lines in every type
PRODUCTS = [("fp4", None, 2100, 2048, 256), ("fp4", None, 5000, 2048, 256), ("fp4", None, 4000, 4096, 256), ("fp8", None, 2100, 2048, 256),
            ("fp8", None, 5000, 2048, 256), ("fp8", None, 4000, 4096, 256), ("fp8", False, 2100, 2048, 300)]


@pytest.mark.parametrize("out_dtype,res_dtype,act", [(torch.float16, None, 1), (torch.bfloat16, torch.bfloat16, 0), (torch.float32, torch.float32, 2),
                                                     (torch.float16, torch.float32, 0)])
@pytest.mark.parametrize("fa,cut,m,n,k", PRODUCTS)
def test_products_of_whole_lines(cuda, fa, cut, m, n, k, out_dtype, res_dtype, act):
    """Into a matrix of its own, in place, and into a window of a wider matrix whose surroundings stay.  A window off the lines takes the
    ordinary stores: the same bits."""
    from crowdsam_amd import hip
    a, w = operands(m, n, k, fa, m + k)
    qa, qw = hip.mx_quantize(a.to(cuda), fa), hip.mx_quantize(w.to(cuda), "fp4")
    bias = torch.randn(n, generator=gen(2)).to(cuda)
    res = None if res_dtype is None else torch.randn(m, n, generator=gen(3)).to(res_dtype).to(cuda)
    kw = dict(bias=bias, act=act, cut=cut)
    out = hip.mx_gemm(qa, qw, residual=res, out_dtype=out_dtype, **kw)
    va, vw = mx_ref.values(qa).to(cuda), mx_ref.values(qw).to(cuda)
    c, tol = va @ vw.t().contiguous(), 2 * U * k * (va.abs() @ vw.abs().t().contiguous())
    if fa == "fp8" and cut is None and out_dtype != torch.float32:
        tol = tol + 15 * 2.0 ** -13 * (group_max(va) @ group_max(vw).t().contiguous())
    c = c + bias.double()
    tol = tol + U * c.abs()
    if act == 1:
        c = c * 0.5 * torch.special.erfc(-c / 2 ** 0.5)
        tol = 1.13 * tol + (6e-6 + 2 * U) * c.abs() + 1.3e-9
    elif act == 2:
        c = c.clamp(min=0)
    if res is not None:
        c = c + res.double()
        tol = tol + U * c.abs()
    f = torch.finfo(out_dtype)
    tol = (tol + f.eps / 2 * c.abs() + f.smallest_normal * f.eps) * (1 + 2.0 ** -7)
    assert bool(((out.double() - c).abs() <= tol).all())
    del c, tol
    if res_dtype == out_dtype:
        x = res.clone()
        assert hip.mx_gemm(qa, qw, residual=x, out=x, **kw).data_ptr() == x.data_ptr() and torch.equal(x, out)
    for width, at in ((n + 128, 64), (n + 4, 1)):          # on the lines of 128 bytes in every type, and off them
        big = torch.full((m + 2, width), 7.0, dtype=out_dtype, device=cuda)
        hip.mx_gemm(qa, qw, residual=res, out=big[1:m + 1, at:at + n], **kw)
        assert torch.equal(big[1:m + 1, at:at + n], out)
        big[1:m + 1, at:at + n] = 7.0
        assert bool((big == 7.0).all())


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("dtype", DTS)
def test_quantised_operands_over_the_caches(cuda, fmt, dtype):
    from crowdsam_amd import hip
    m, k = (30003, 2112) if fmt == "fp4" else (15001, 2112)
    g = torch.Generator(device=cuda).manual_seed(5)
    x = (torch.randn(m, k, device=cuda, generator=g) * torch.exp2(torch.randint(-9, 9, (m, 1), device=cuda, generator=g).float())).to(dtype)
    q = hip.mx_quantize(x, fmt)
    assert m * q.codes.shape[1] > 32 << 20
    for i in range(0, m, 7000):                            # (too small for it)
        p = hip.mx_quantize(x[i:i + 7000], fmt)
        assert torch.equal(q.codes[i:i + 7000], p.codes) and torch.equal(q.scales[:, i:i + 7000], p.scales)
    rows = torch.cat((torch.arange(100), torch.arange(m - 100, m)))
    codes, scales = mx_ref.quantize(x[rows.to(cuda)].cpu(), fmt)
    assert torch.equal(q.codes[rows.to(cuda)].cpu(), codes) and torch.equal(q.scales[:, rows.to(cuda)].cpu(), scales)


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("dtype", DTS)
def test_dequantised_rows_over_the_caches(cuda, fmt, dtype):
    from crowdsam_amd import hip
    m, k = 8301, 2112                                      # rows of whole lines in every type, the last segment of 256 part-filled
    q = hip.mx_quantize(torch.randn(m, k, generator=gen(6)).to(cuda), fmt)
    y = hip.mx_dequantize(q, out_dtype=dtype)
    assert y.numel() * y.element_size() > 32 << 20
    v = mx_ref.values(q)
    assert equal(y.cpu(), v.float().to(dtype))


@pytest.mark.parametrize("dtype,res,out_dtype,m,d", [(torch.bfloat16, torch.bfloat16, torch.bfloat16, 66003, 1024), (torch.float16, torch.float32, "fp8", 53001, 1040),
                                                     (torch.float16, torch.float32, "fp4", 66001, 1024), (torch.bfloat16, None, torch.float32, 66001, 1024),
                                                     (torch.float32, torch.float32, torch.float16, 45001, 1024), (torch.float16, None, torch.float16, 66001, 2176),
                                                     (torch.float16, torch.float16, torch.float32, 5501, 8320), (torch.float32, None, torch.float32, 2101, 32768),
                                                     (torch.bfloat16, torch.bfloat16, torch.bfloat16, 66003, 1025), (torch.float16, torch.float32, "fp8", 53001, 1031)])
def test_normed_rows_over_the_caches(cuda, dtype, res, out_dtype, m, d):
    from crowdsam_amd import hip
    g = torch.Generator(device=cuda).manual_seed(d)
    x = (torch.randn(m, d, device=cuda, generator=g) + 0.5).to(dtype)
    gamma = torch.rand(d, device=cuda, generator=g) + 0.5
    r = None if res is None else torch.randn(m, d, device=cuda, generator=g).to(res)

    def norm(i, j):
        y = hip.rms_norm(x[i:j], gamma, EPS, residual=None if r is None else r[i:j], out_dtype=out_dtype)
        return (y, None) if r is None else y

    y, h = norm(0, m)
    step = -(-m // 4)
    for i in range(0, m, step):
        p, q = norm(i, i + step)                           # (too small for it)
        if out_dtype in ("fp8", "fp4"):
            assert torch.equal(y.codes[i:i + step], p.codes) and torch.equal(y.scales[:, i:i + step], p.scales)
        else:
            assert torch.equal(y[i:i + step], p)
        assert r is None or torch.equal(h[i:i + step], q)
    for i in range(0, m, 8192):                            # 40 fp32 steps, as test_rms_norm_gpu counts them, and the store's rounding
        s = x[i:i + 8192].double() if r is None else x[i:i + 8192].double() + r[i:i + 8192].double()
        if r is not None:
            f = torch.finfo(res)
            assert bool(((h[i:i + 8192].double() - s).abs() <= s.abs() * (U + f.eps / 2) * (1 + 2.0 ** -7) + f.smallest_normal * f.eps).all())
        if out_dtype in DTS:
            f = torch.finfo(out_dtype)
            ref = s / torch.sqrt(s.square().mean(1, keepdim=True) + EPS) * gamma.double()
            assert bool(((y[i:i + 8192].double() - ref).abs() <= ref.abs() * (40 * U + f.eps / 2) * (1 + 2.0 ** -7) + f.smallest_normal * f.eps).all())
    if out_dtype in ("fp8", "fp4"):                        # the fp32 row, then the definition of the format
        last = hip.rms_norm(x[-200:], gamma, EPS, out_dtype=torch.float32) if r is None else \
            hip.rms_norm(x[-200:], gamma, EPS, residual=r[-200:], out_dtype=torch.float32)[0]
        codes, scales = mx_ref.quantize(last.cpu(), out_dtype)
        assert torch.equal(y.codes[-200:].cpu(), codes) and torch.equal(y.scales[:, -200:].cpu(), scales)


@pytest.mark.parametrize("dtype", DTS)
@pytest.mark.parametrize("T,Hq,Hk,hd,sections,interleaved", [(4201, 20, 12, 128, (32, 32), False), (4201, 32, 0, 128, (16, 16), False), (8401, 24, 8, 64, (16, 16), True),
                                                            (7001, 16, 16, 80, (12, 14, 14), True), (15001, 24, 8, 36, (9, 8), True),
                                                            (7001, 16, 16, 80, (20, 20), False), (6001, 24, 8, 97, (40,), True)])
def test_rotated_rows_over_the_caches(cuda, dtype, T, Hq, Hk, hd, sections, interleaved):
    from crowdsam_amd import hip
    g = torch.Generator(device=cuda).manual_seed(T)
    x = torch.randn(T, (Hq + Hk) * hd, device=cuda, generator=g).to(dtype)
    q = x[:, :Hq * hd].unflatten(1, (Hq, hd))
    k = x[:, Hq * hd:].unflatten(1, (Hk, hd)) if Hk else None
    freq, axis = hip.rotary_frequencies(sections)
    pos = positions(len(sections), T, torch.float32, hd).to(cuda)
    assert x.numel() * x.element_size() > 32 << 20
    outs = hip.rotary(q, k, pos, freq, axis, interleaved=interleaved)
    for i in range(0, T, 1500):                            # (too small for it)
        part = hip.rotary(q[i:i + 1500], None if k is None else k[i:i + 1500], pos[:, i:i + 1500].contiguous(), freq, axis, interleaved=interleaved)
        for a, b in zip(outs, part):
            assert a is None or torch.equal(a[i:i + 1500], b)
    for i in (0, T - 60):
        for a, b in zip(outs, (q, k)):
            if a is not None:
                check_rotary(a[i:i + 60], b[i:i + 60].cpu(), pos[:, i:i + 60].cpu(), freq.cpu(), axis.cpu(), interleaved)
    before = [t.clone() for t in outs if t is not None]
    hip.rotary(q, k, pos, freq, axis, interleaved=interleaved, q_out=q, k_out=k)                  # in place
    for a, b in zip((q, k), before):
        assert torch.equal(a, b)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTS)
def test_rotated_rows_into_windows(cuda, dtype, interleaved):
    """Windows on the lines of 128 bytes and off them, by the column, by the row pitch and by k alone: the same bits, the rest untouched."""
    from crowdsam_amd import hip
    T, H, hd = 4201, 16, 128
    x = torch.randn(T, 2 * H * hd, generator=gen(9)).to(dtype).to(cuda)
    q, k = (x[:, i * H * hd:(i + 1) * H * hd].unflatten(1, (H, hd)) for i in range(2))
    freq, axis = hip.rotary_frequencies((32, 32))
    pos = positions(2, T, torch.int32, hd).to(cuda)
    want = hip.rotary(q, k, pos, freq, axis, interleaved=interleaved)
    for width, q_at, k_at in ((2 * H * hd + 128, 64, 64 + H * hd), (2 * H * hd + 128, 3, 3 + H * hd), (2 * H * hd + 7, 0, H * hd),
                              (2 * H * hd + 128, 0, H * hd + 8)):
        big = torch.full((T, width), 5.0, dtype=dtype, device=cuda)
        views = [big[:, at:at + H * hd].unflatten(1, (H, hd)) for at in (q_at, k_at)]
        hip.rotary(q, k, pos, freq, axis, interleaved=interleaved, q_out=views[0], k_out=views[1])
        for v, w in zip(views, want):
            assert torch.equal(v, w)
            v.fill_(5.0)
        assert bool((big == 5.0).all())
