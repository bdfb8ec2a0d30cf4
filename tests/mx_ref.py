"""Plain CPU forms of the microscaled format in float64, written from its definition; used by the tests only."""
import torch

FP4 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
FP8 = torch.tensor([(m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127],
                   dtype=torch.float64)
EMAX = {"fp4": 2, "fp8": 8}


def padded(k):
    return -(-k // 256) * 256


def quantize(x, fmt):
    """(codes, scales) of the rows of ``x`` in the layout of hip.MxTensor."""
    grid = FP4 if fmt == "fp4" else FP8
    m, k = x.shape
    b = torch.zeros(m, padded(k), dtype=torch.float64)
    b[:, :k] = x.double().cpu()
    sign = torch.zeros(m, padded(k), dtype=torch.bool)
    sign[:, :k] = torch.signbit(x.cpu())
    b = b.view(m, -1, 32)
    bad = ~torch.isfinite(b).all(2)
    amax = b.abs().amax(2)
    amax[bad] = 1.0
    e = torch.full_like(amax, -127)
    normal = amax >= 2.0 ** -126
    f, ex = torch.frexp(amax[normal])                       # amax = f 2^ex, f in [1/2, 1)
    e[normal] = (ex - 1 - EMAX[fmt]).clamp(min=-127).double()
    a = (b / torch.exp2(e)[..., None]).abs()
    a[bad] = 0
    mid = (grid[1:] + grid[:-1]) / 2
    lo, hi = torch.searchsorted(mid, a), torch.searchsorted(mid, a, right=True)
    code = torch.where(hi % 2 == 0, hi, lo)                 # on a tie the two differ by one: the even one
    code = (code + sign.view_as(code) * 8 if fmt == "fp4" else code + sign.view_as(code) * 128).to(torch.uint8)
    code[bad] = 0
    code = code.view(m, -1)
    if fmt == "fp4":
        code = code[:, 0::2] | (code[:, 1::2] << 4)
    s = (e + 127).to(torch.uint8)
    s[bad] = 255
    return code, s.view(m, -1, 4).transpose(0, 1).contiguous()


def values(q):
    """float64 [rows, K] of an hip.MxTensor."""
    codes, scales = q.codes.cpu().long(), q.scales.cpu().double()
    if q.fmt == "fp4":
        codes = torch.stack((codes & 15, codes >> 4), 2).flatten(1)
        v = torch.cat((FP4, -FP4))[codes]
    else:
        g = torch.cat((FP8, torch.tensor([float("nan")], dtype=torch.float64)))
        v = torch.cat((g, -g))[codes]
    s = torch.where(scales == 255, torch.nan, torch.exp2(scales - 127)).transpose(0, 1).flatten(1)
    return (v * s.repeat_interleave(32, 1))[:, :q.K]
