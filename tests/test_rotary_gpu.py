"""hip.rotary against float64."""
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(x, pos, freq, axis, interleaved):
    """(result, sum of the magnitudes that enter it) in float64."""
    P = freq.numel()
    T = x.shape[0]
    i = torch.arange(P) * (2 if interleaved else 1)
    j = i + (1 if interleaved else P)
    ang = pos.double()[axis.long()].t() * freq
    ang = ang.repeat(T // pos.shape[1], 1)[:, None]
    y = x.double().clone()
    mag = torch.zeros_like(y)
    a, b = x.double()[..., i], x.double()[..., j]
    y[..., i], y[..., j] = a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()
    mag[..., i] = mag[..., j] = a.abs() + b.abs()
    return y, mag


def check(out, x, pos, freq, axis, interleaved):
    """cos and sin: the angle in turns is rounded once to fp32 (pi U of the angle at most), the function to an ulp, then two products and
    a sum: 8 U of |a| + |b| cover it; then the store rounds.  What passes through is the same bits."""
    ref, mag = reference(x, pos, freq, axis, interleaved)
    out = out.cpu()
    f = torch.finfo(out.dtype)
    tol = 8 * U * mag + (f.eps / 2 * ref.abs() + f.smallest_normal * f.eps) * (mag > 0)
    tol = tol * (1 + 2.0 ** -7)
    d = (out.double() - ref).abs()
    assert bool((d <= tol).all()), float((d - tol).max())
    P = 2 * freq.numel()
    assert torch.equal(out[..., P:], x[..., P:])


def positions(A, T, kind, seed):
    g = torch.Generator().manual_seed(seed)
    far = torch.tensor([2.0 ** 20, 1024.0, 64.0])[:A, None]
    p = (torch.rand(A, T, generator=g) * 2 - 1) * far
    return p.to(torch.int32) if kind == torch.int32 else p


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,Hq,Hk,hd,sections", [(1, 16, 16, 64, (16, 16)), (1, 1, 0, 2, (1,)), (5, 3, 1, 80, (12, 14, 14)), (70, 4, 4, 80, (12, 12, 12)),
                                                 (33, 2, 1, 64, (8,)), (17, 5, 2, 36, (9, 8)), (9, 24, 6, 128, (16, 24, 24)), (3, 2, 2, 250, (60, 50)),
                                                 (258, 1, 1, 16, (4, 4)), (4, 3, 0, 7, (2, 1)), (13, 20, 0, 250, (23,)), (9, 5, 5, 250, (20, 20, 13)),
                                                 (40, 18, 18, 36, (11,)), (6, 2, 2, 97, (7, 8)), (5, 1, 2, 31, (15,)), (2000, 24, 24, 250, (61, 62)), (3, 2, 1, 4096, (1024, 1024)),
                                                 (2, 1, 1, 4095, (2047,))])
def test_matches_float64(cuda, dtype, interleaved, T, Hq, Hk, hd, sections):
    from crowdsam_amd import hip
    g = torch.Generator().manual_seed(T + hd)
    x = torch.randn(T, (Hq + 2 * Hk) * hd, generator=g).to(dtype)
    freq, axis = hip.rotary_frequencies(sections, device="cpu")
    for kind in (torch.int32, torch.float32):
        pos = positions(len(sections), T, kind, hd)
        d = x.to(cuda)
        q, k = d[:, :Hq * hd].unflatten(1, (Hq, hd)), d[:, Hq * hd:(Hq + Hk) * hd].unflatten(1, (Hk, hd)) if Hk else None
        qo, ko = hip.rotary(q, k, pos.to(cuda), freq.to(cuda), axis.to(cuda), interleaved)
        check(qo, x[:, :Hq * hd].unflatten(1, (Hq, hd)), pos, freq, axis, interleaved)
        if Hk:
            check(ko, x[:, Hq * hd:(Hq + Hk) * hd].unflatten(1, (Hk, hd)), pos, freq, axis, interleaved)
        else:
            assert ko is None
        assert torch.equal(d.cpu(), x)
        # in place in the qkv matrix: the same bits, and v untouched
        hip.rotary(q, k, pos.to(cuda), freq.to(cuda), axis.to(cuda), interleaved, q_out=q, k_out=k)
        assert torch.equal(q, qo) and (k is None or torch.equal(k, ko)) and torch.equal(d[:, (Hq + Hk) * hd:].cpu(), x[:, (Hq + Hk) * hd:])


def test_shared_positions_head_major_and_unaligned(cuda):
    from crowdsam_amd import hip
    g = torch.Generator().manual_seed(1)
    freq, axis = hip.rotary_frequencies((10, 10), device="cpu")
    pos = positions(2, 30, torch.int32, 4)
    x = torch.randn(5, 90, 48, generator=g).half()                   # [heads, tokens, hd]
    xt = x.transpose(0, 1)
    out, _ = hip.rotary(x.to(cuda).transpose(0, 1), None, pos.to(cuda), freq.to(cuda), axis.to(cuda))
    check(out, xt, pos, freq, axis, False)                           # three images of 30 positions
    y = torch.randn(30, 5 * 48 + 1, generator=g).half()
    z = y[:, 1:].unflatten(1, (5, 48))
    out, _ = hip.rotary(y.to(cuda)[:, 1:].unflatten(1, (5, 48)), None, pos.to(cuda), freq.to(cuda), axis.to(cuda))
    check(out, z, pos, freq, axis, False)
    wide = torch.zeros(2, 64, dtype=torch.int32)
    wide[:, 3:33] = pos
    out2, _ = hip.rotary(y.to(cuda)[:, 1:].unflatten(1, (5, 48)), None, wide.to(cuda)[:, 3:33], freq.to(cuda), axis.to(cuda))
    assert torch.equal(out, out2)


def test_gradient_is_the_call_with_negated_positions(cuda):
    """<dy, f(x)> is linear in x: its derivative along e is <dy, f(e)>, taken as a difference of f, and the adjoint gives <f*(dy), e>."""
    from crowdsam_amd import hip
    g = torch.Generator().manual_seed(2)
    freq, axis = hip.rotary_frequencies((12, 12, 8))
    pos = positions(3, 20, torch.float32, 1).to(cuda)
    x, e, dy = (torch.randn(20, 3, 80, generator=g).to(cuda) for _ in range(3))
    f = lambda v, p: hip.rotary(v, None, p, freq, axis)[0].double()  # noqa: E731
    step = 2.0 ** -4
    diff = ((f(x + step * e, pos) - f(x - step * e, pos)) / (2 * step) * dy.double()).sum()
    adj = (f(dy, -pos) * e.double()).sum()
    # |f(x +- s e)| is off by 8 U (|a| + |b|) <= 8 U 2 (|x| + |e|) at most, over 2 s, and the sums x +- s e round too
    bound = (16 * U * 2 * (x.abs().double() + e.abs().double()).amax() / (2 * step) * dy.abs().double().sum() * 2) + 16 * U * (dy.abs() * e.abs()).double().sum() * 4
    assert abs(float(diff - adj)) <= float(bound)
    ang = (pos.double()[axis.long()].t() * freq)[:, None]
    want = dy.double().clone()
    a, b = dy.double()[..., :32], dy.double()[..., 32:64]
    want[..., :32], want[..., 32:64] = a * ang.cos() + b * ang.sin(), -a * ang.sin() + b * ang.cos()
    assert float((f(dy, -pos) - want).abs().max()) <= 16 * U * 2 * float(dy.abs().max())


def test_graph_replays(cuda):
    from crowdsam_amd import hip
    freq, axis = hip.rotary_frequencies((16, 16))
    x = torch.randn(40, 4, 64, device=cuda).half()
    pos = torch.randint(0, 1000, (2, 40), dtype=torch.int32, device=cuda)
    hip.rotary(x, None, pos, freq, axis)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, _ = hip.rotary(x, None, pos, freq, axis)
    for _ in range(4):
        pos.add_(3)
        x.neg_()
        fresh = hip.rotary(x, None, pos, freq, axis)[0].clone()
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, fresh)
