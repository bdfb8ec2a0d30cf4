"""The low-precision operators together, as a pre-norm encoder block over the tokens of two images uses them around the framework's flash
attention: every call works on what the call before it wrote, and is held to its own definition in float64 on those inputs."""
import pytest
import torch

import mx_ref
from test_mx_gpu import close, gen, product_ref
from test_rms_norm_gpu import EPS, check as check_norm
from test_rotary_gpu import check as check_rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("side,images", [(1, 1), (9, 2)])
def test_encoder_block(cuda, side, images):
    from crowdsam_amd import hip
    D, nH, hidden = 256, 4, 640
    T = side * side
    rows = T * images
    g = gen(side)

    def weight(n, k):
        return hip.mx_quantize((torch.randn(n, k, generator=g) / k ** 0.5).to(cuda), "fp4")

    x = (torch.randn(rows, D, generator=g) + 3 * torch.randn(D, generator=g)).to(cuda)              # fp32 residual stream
    g1, g2 = ((torch.rand(D, generator=g) + 0.5).to(cuda) for _ in range(2))
    b_qkv, b_proj, b1, b2 = (0.1 * torch.randn(n, generator=g).to(cuda) for n in (3 * D, D, hidden, D))
    w_qkv, w_proj, w1, w2 = weight(3 * D, D), weight(D, D), weight(hidden, D), weight(D, hidden)
    freq, axis = hip.rotary_frequencies((16, 16))
    yy, xx = torch.meshgrid(torch.arange(side), torch.arange(side), indexing="ij")
    pos = torch.stack((yy.flatten(), xx.flatten())).to(torch.int32).to(cuda)

    def normed(y, h, gamma):
        ref = h.double() / torch.sqrt(h.double().square().mean(1, keepdim=True) + EPS) * gamma.double()
        f32 = hip.rms_norm(h, gamma, EPS, out_dtype=torch.float32)
        check_norm(f32, ref.cpu(), torch.float32, 40)
        codes, scales = mx_ref.quantize(f32, "fp8")
        assert torch.equal(y.codes.cpu(), codes) and torch.equal(y.scales.cpu(), scales)

    n1 = hip.rms_norm(x, g1, EPS, out_dtype="fp8")
    normed(n1, x, g1)
    qkv = hip.mx_gemm(n1, w_qkv, bias=b_qkv)
    close(qkv, *product_ref(hip, n1, w_qkv, b_qkv.cpu(), 0, None, torch.float16))
    q, k = (qkv[:, i * D:(i + 1) * D].unflatten(1, (nH, 64)) for i in range(2))
    before = qkv.cpu()
    hip.rotary(q, k, pos, freq, axis, q_out=q, k_out=k)
    for got, i in ((q, 0), (k, 1)):
        check_rotary(got, before[:, i * D:(i + 1) * D].unflatten(1, (nH, 64)), pos.cpu(), freq.cpu(), axis.cpu(), False)
    assert torch.equal(qkv[:, 2 * D:].cpu(), before[:, 2 * D:])
    att = torch.empty(rows, D, dtype=torch.float16, device=cuda)
    hip.flash_attn(qkv, att, T, nH, 0.125, D, n_images=images)
    qkv64 = qkv.cpu().double().view(images, T, 3, nH, 64).permute(2, 0, 3, 1, 4)
    ref = (torch.softmax(qkv64[0] @ qkv64[1].transpose(-1, -2).contiguous() * 0.125, -1) @ qkv64[2]).transpose(1, 2).reshape(rows, D)
    # softmax weights and v in fp16 (2^-11 each), the output in fp16; scores to 2^-10 of their size
    assert float((att.cpu().double() - ref).abs().max()) < 4e-3 * float(qkv64[2].abs().max())
    a8 = hip.mx_quantize(att, "fp8")
    x0 = x.cpu()
    hip.mx_gemm(a8, w_proj, bias=b_proj, out=x, residual=x)
    close(x, *product_ref(hip, a8, w_proj, b_proj.cpu(), 0, x0, torch.float32))
    n2 = hip.rms_norm(x, g2, EPS, out_dtype="fp8")
    normed(n2, x, g2)
    h = hip.mx_gemm(n2, w1, bias=b1, act=hip.ACT_GELU)
    close(h, *product_ref(hip, n2, w1, b1.cpu(), hip.ACT_GELU, None, torch.float16))
    h4 = hip.mx_quantize(h, "fp4")
    codes, scales = mx_ref.quantize(h, "fp4")
    assert torch.equal(h4.codes.cpu(), codes) and torch.equal(h4.scales.cpu(), scales)
    x1 = x.cpu()
    out = hip.mx_gemm(h4, w2, bias=b2, residual=x, out=x)
    assert out.data_ptr() == x.data_ptr()
    close(out, *product_ref(hip, h4, w2, b2.cpu(), 0, x1, torch.float32))
