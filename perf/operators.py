"""Measured cases of the low-precision encoder-block operators: root-mean-square norm with the residual's addition
(``hip.rms_norm``), microscaled quantisation (``hip.mx_quantize`` / ``hip.mx_dequantize``), the product of microscaled operands
(``hip.mx_gemm``) and rotary positions with several axes (``hip.rotary``).

``run`` computes a case in its plain form (elementary torch operations in 32 bits) or, where ``own`` is true, with the calls a
user makes.  Microscaled operands are the layout the framework documents: codes uint8 [rows, Kp / 2] (E2M1, element 2i in the low
nibble) or [rows, Kp] (E4M3), scales uint8 [Kp / 128, rows, 4] (E8M0, the scale of block b of row r at [b / 4, r, b % 4]), Kp = K
rounded up to a multiple of 256, zero codes behind K.
"""
import math

import torch

own = False

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"f16": 2, "bf16": 2, "f32": 4, "fp8": 1, "fp4": 0.5}
EMAX = {"fp4": 2, "fp8": 8}
TOP = {"fp4": 6.0, "fp8": 448.0}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
EPS = 1e-6


def padded(k):
    return -(-k // 256) * 256


# ---------------------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token's row between two projections of a streamed pass: the call's latency
        dict(name="norm one token", op="norm", rows=1, width=1024, x="f16", res="f32", out="fp8"),
        # DINOv2 ViT-L rows of one frame (73 x 73 patches + the class token), fp32 residual stream, 8-bit operand of the qkv product
        dict(name="norm one frame", op="norm", rows=5330, width=1024, x="f16", res="f32", out="fp8"),
        # sixteen ViT-H frames of 64 x 64 tokens, everything bfloat16
        dict(name="norm sixteen frames", op="norm", rows=65536, width=1280, x="bf16", res="bf16", out="bf16"),
        # a ViT-H fc1 weight laid out at load time, and read back to look at what 4 bits cost it
        dict(name="quantise weight 4 bit", op="quant", rows=5120, width=1280, x="f32", fmt="fp4"),
        # the fc2 operand of four DINOv2 frames
        dict(name="quantise activations 8 bit", op="quant", rows=21320, width=4096, x="f16", fmt="fp8"),
        # a ragged little operand: a row pitch and a width that are multiples of nothing
        dict(name="quantise ragged", op="quant", rows=333, width=1001, x="bf16", fmt="fp4"),
        # one token through a fc1: every weight read for one row
        dict(name="product one token", op="gemm", rows=1, cols=4096, width=1024, a="fp8", bias=True, act="gelu", res="none", out="f16"),
        # the seven tokens of 32 prompts: few tiles
        dict(name="product prompt tokens", op="gemm", rows=224, cols=2048, width=1024, a="fp4", bias=True, act="relu", res="none", out="f16"),
        # fc1 of one DINOv2 frame, 8-bit activations
        dict(name="product one frame", op="gemm", rows=5330, cols=4096, width=1024, a="fp8", bias=True, act="gelu", res="none", out="f16"),
        # fc2-sized product of four DINOv2 frames onto the fp32 residual stream, 4 bits on both sides
        dict(name="product four frames", op="gemm", rows=21320, cols=4096, width=4096, a="fp4", bias=True, act="none", res="f32", out="f32"),
        # one token's heads
        dict(name="rotary one token", op="rotary", tokens=1, images=1, heads=16, kv=16, dim=64, axes=2, pairs=32, half=True, x="f16", pos="i32"),
        # four frames of a clip, (time, height, width) positions, 2 x 16 heads of 80 out of the qkv matrix
        dict(name="rotary clip", op="rotary", tokens=16384, images=1, heads=16, kv=16, dim=80, axes=3, pairs=36, half=False, x="f16", pos="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("norm", "quant", "gemm", "gemm", "rotary"))
    if op == "norm":
        rows, width = _log(rng, 1, 65536), _log(rng, 32, 8192)
        rows = min(rows, max(1, 65536 * 1280 // (2 * width)))
        x = rng.choice(("f16", "bf16", "f32"))
        return dict(op=op, rows=rows, width=width, x=x, res=rng.choice(("none", x, "f32")),
                    out=rng.choice(("f16", "bf16", "f32", "fp8", "fp4")))
    if op == "quant":
        rows, width = _log(rng, 1, 65536), _log(rng, 32, 16384)
        rows = min(rows, max(1, 21320 * 4096 // (2 * width)))
        return dict(op=op, rows=rows, width=width, x=rng.choice(("f16", "bf16", "f32")), fmt=rng.choice(("fp4", "fp8")))
    if op == "gemm":
        rows, cols, width = _log(rng, 1, 32768), _log(rng, 16, 8192), _log(rng, 32, 8192)
        if rng.random() < 0.5:
            cols, width = -(-cols // 128) * 128, padded(width)
        rows = min(rows, max(1, 21320 * 4096 * 4096 // (2 * cols * width)), max(1, 21320 * 4096 // (2 * cols)))
        out = rng.choice(("f16", "bf16", "f32"))
        return dict(op=op, rows=rows, cols=cols, width=width, a=rng.choice(("fp8", "fp4")), bias=rng.random() < 0.7,
                    act=rng.choice(("none", "gelu", "relu")), res=rng.choice(("none", out, "f32")), out=out)
    axes = rng.choice((1, 2, 3))
    dim = rng.choice((16, 32, 64, 80, 96, 128, 36, 250))
    pairs = rng.randint(axes, dim // 2)
    heads = rng.randint(1, 24)
    kv = rng.choice((0, 1, heads, max(1, heads // 4)))
    images = rng.choice((1, 1, 2, 4))
    tokens = _log(rng, 1, 32768)
    tokens = min(tokens, max(1, 16384 * 32 * 80 // (2 * images * (heads + kv) * dim)))
    return dict(op=op, tokens=tokens, images=images, heads=heads, kv=kv, dim=dim, axes=axes, pairs=pairs, half=rng.random() < 0.5,
                x=rng.choice(("f16", "bf16", "f32")), pos=rng.choice(("i32", "f32")))


# --------------------------------------------------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _rows(m, k, g, dtype):
    """Rows of a residual stream: unit noise, a common offset per channel, and a few channels that are far larger."""
    x = torch.randn(m, k, generator=g, device="cuda")
    ch = torch.randn(k, generator=g, device="cuda") * 0.3
    ch[torch.randint(0, k, (max(1, k // 256),), generator=g, device="cuda")] += 30.0
    return (x + ch).to(dtype)


def _operand(m, k, g, fmt, spread):
    """A microscaled operand of gaussian rows, as the framework lays it out."""
    return _mx_pack(torch.randn(m, k, generator=g, device="cuda") * spread, fmt)


def _frequencies(case):
    """Radians per unit of position and the axis of every pair: the pairs are dealt out to the axes in equal runs, and each axis
    has its own geometric spectrum."""
    p, a = case["pairs"], case["axes"]
    axis = [i * a // p for i in range(p)]
    freq = []
    for ax in range(a):
        n = axis.count(ax)
        freq += [10000.0 ** (-i / n) for i in range(n)]
    return torch.tensor(freq, dtype=torch.float64, device="cuda"), torch.tensor(axis, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    if op == "norm":
        m, d = case["rows"], case["width"]
        s = dict(case=case, x=_rows(m, d, g, DT[case["x"]]), gamma=torch.rand(d, generator=g, device="cuda") + 0.5, residual=None)
        if case["res"] != "none":
            s["residual"] = _rows(m, d, g, DT[case["res"]])
        return s
    if op == "quant":
        return dict(case=case, x=_rows(case["rows"], case["width"], g, DT[case["x"]]))
    if op == "gemm":
        m, n, k = case["rows"], case["cols"], case["width"]
        s = dict(case=case, bias=None, residual=None)
        s["a"], s["a_scales"] = _operand(m, k, g, case["a"], 1.0)
        s["w"], s["w_scales"] = _operand(n, k, g, "fp4", 1.0 / math.sqrt(k))
        if case["bias"]:
            s["bias"] = torch.randn(n, generator=g, device="cuda") * 0.1
        if case["res"] != "none":
            s["residual"] = torch.randn(m, n, generator=g, device="cuda").to(DT[case["res"]])
        return s
    t = case["tokens"]
    width = (case["heads"] + 2 * max(case["kv"], 1)) * case["dim"]
    # the token-major output of a qkv projection: q, k and v side by side
    qkv = torch.randn(t * case["images"], width, generator=g, device="cuda").to(DT[case["x"]])
    q = qkv[:, :case["heads"] * case["dim"]].unflatten(1, (case["heads"], case["dim"]))
    k = None
    if case["kv"]:
        k = qkv[:, case["heads"] * case["dim"]:(case["heads"] + case["kv"]) * case["dim"]].unflatten(1, (case["kv"], case["dim"]))
    far = torch.tensor([100000, 1024, 1024][:case["axes"]], device="cuda")[:, None]      # a long clip's times, a frame's rows and columns
    if case["pos"] == "i32":
        pos = (torch.rand(case["axes"], t, generator=g, device="cuda") * far).to(torch.int32)
    else:
        pos = torch.rand(case["axes"], t, generator=g, device="cuda") * far
    freq, axis = _frequencies(case)
    return dict(case=case, q=q, k=k, pos=pos, freq=freq, axis=axis)


# ---------------------------------------------------------------------------------------------------------- plain forms
def _mx_blocks(x, fmt):
    """(rounded values in units of their scale [m, blocks, 32], exponents [m, blocks]) of fp32 rows, padded."""
    m, k = x.shape
    b = torch.zeros(m, padded(k), dtype=torch.float32, device=x.device)
    b[:, :k] = x
    b = b.view(m, -1, 32)
    amax = b.abs().amax(2)
    e = (torch.frexp(amax).exponent - 1 - EMAX[fmt]).clamp(-127, 127)
    e = torch.where(amax < 2.0 ** -126, torch.full_like(e, -127), e)
    # two exact steps: one power of two of the whole range has no fp32 value
    half = torch.div(-e, 2, rounding_mode="floor")
    v = b * torch.exp2(half.float())[..., None] * torch.exp2((-e - half).float())[..., None]
    a = v.abs().clamp(max=TOP[fmt])
    if fmt == "fp4":
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    else:
        step = torch.exp2((torch.frexp(a).exponent - 4).clamp(min=-9).float())      # 2^(floor(log2 a) - 3), subnormals 2^-9
    r = (torch.round(a / step) * step).clamp(max=TOP[fmt])       # torch.round: ties to even
    return torch.copysign(r, v), e


def _mx_scales(e):
    """E8M0 bytes of exponents [m, blocks], in the operand's order."""
    return (e + 127).to(torch.uint8).view(e.shape[0], -1, 4).transpose(0, 1).contiguous()


def _mx_pack(x, fmt):
    """(codes, scales) of fp32 rows."""
    v, e = _mx_blocks(x, fmt)
    scales = _mx_scales(e)
    if fmt == "fp8":
        return v.view(x.shape[0], -1).to(torch.float8_e4m3fn).view(torch.uint8), scales
    a = v.abs()
    code = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code = (code | (torch.signbit(v).to(torch.uint8) << 3)).view(x.shape[0], -1)
    return code[:, 0::2] | (code[:, 1::2] << 4), scales


def _mx_values(codes, scales, fmt):
    """fp32 values of a microscaled operand."""
    if fmt == "fp8":
        v = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=codes.device)
        v = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), 2)
    v = v.view(codes.shape[0], -1, 32)
    e = scales.float().transpose(0, 1).reshape(codes.shape[0], -1) - 127
    return (v * torch.exp2(e)[..., None]).view(codes.shape[0], -1)


def _mx_out(x, fmt):
    """What a quantising call hands back: 8-bit codes as they are, 4-bit ones as the values they stand for."""
    v, e = _mx_blocks(x, fmt)
    scales = _mx_scales(e).view(torch.float8_e8m0fnu)
    if fmt == "fp8":
        return {"codes": v.view(x.shape[0], -1).to(torch.float8_e4m3fn), "scales": scales}
    return {"values": (v * torch.exp2(e.float())[..., None]).view(x.shape[0], -1)[:, :x.shape[1]].to(torch.bfloat16), "scales": scales}


def _plain(s):
    case = s["case"]
    op = case["op"]
    if op == "norm":
        h = s["x"].float()
        if s["residual"] is not None:
            h = h + s["residual"].float()
        y = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["gamma"]
        out = _mx_out(y, case["out"]) if case["out"] in EMAX else {"y": y.to(DT[case["out"]])}
        if s["residual"] is not None:
            out["h"] = h.to(s["residual"].dtype)
        return out
    if op == "quant":
        return _mx_out(s["x"].float(), case["fmt"])
    if op == "gemm":
        c = _mx_values(s["a"], s["a_scales"], case["a"]) @ _mx_values(s["w"], s["w_scales"], "fp4").t()
        if s["bias"] is not None:
            c = c + s["bias"]
        if case["act"] == "gelu":
            c = 0.5 * c * (1 + torch.erf(c * math.sqrt(0.5)))
        elif case["act"] == "relu":
            c = c.clamp(min=0)
        if s["residual"] is not None:
            c = c + s["residual"].float()
        return c.to(DT[case["out"]])
    p = case["pairs"]
    angle = s["pos"].double()[s["axis"].long()].t() * s["freq"]                          # [tokens, pairs]
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    out = {}
    for name in ("q", "k"):
        if s[name] is None:
            continue
        x = s[name].float().unflatten(0, (case["images"], -1))
        y = x.clone()
        i, j = (slice(0, p), slice(p, 2 * p)) if case["half"] else (slice(0, 2 * p, 2), slice(1, 2 * p, 2))
        y[..., i] = x[..., i] * cos - x[..., j] * sin
        y[..., j] = x[..., i] * sin + x[..., j] * cos
        out[name] = y.flatten(0, 1).to(s[name].dtype)
    return out


# ------------------------------------------------------------------------------------------------- the framework's calls
def _own_mx(hip, q):
    scales = q.scales.view(torch.float8_e8m0fnu)
    if q.fmt == "fp8":
        return {"codes": q.codes.view(torch.float8_e4m3fn), "scales": scales}
    return {"values": hip.mx_dequantize(q, out_dtype=torch.bfloat16), "scales": scales}


def _own(s):
    from crowdsam_amd import hip
    case = s["case"]
    op = case["op"]
    if op == "norm":
        kind = case["out"] if case["out"] in EMAX else DT[case["out"]]
        if s["residual"] is None:
            y, h = hip.rms_norm(s["x"], s["gamma"], EPS, out_dtype=kind), None
        else:
            y, h = hip.rms_norm(s["x"], s["gamma"], EPS, residual=s["residual"], out_dtype=kind)
        out = _own_mx(hip, y) if case["out"] in EMAX else {"y": y}
        if h is not None:
            out["h"] = h
        return out
    if op == "quant":
        return _own_mx(hip, hip.mx_quantize(s["x"], case["fmt"]))
    if op == "gemm":
        k = case["width"]
        act = {"none": hip.ACT_NONE, "gelu": hip.ACT_GELU, "relu": hip.ACT_RELU}[case["act"]]
        return hip.mx_gemm(hip.MxTensor(s["a"], s["a_scales"], case["a"], k), hip.MxTensor(s["w"], s["w_scales"], "fp4", k),
                           bias=s["bias"], act=act, residual=s["residual"], out_dtype=DT[case["out"]])
    q, k = hip.rotary(s["q"], s["k"], s["pos"], s["freq"], s["axis"], interleaved=not case["half"])
    return {"q": q} if k is None else {"q": q, "k": k}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------------------------------ in 64 bits
def _exact_round(v, fmt):
    """The nearest number of the format to every value of `v` (float64), ties to the even code, saturated."""
    if fmt == "fp4":
        grid = torch.tensor(E2M1, dtype=torch.float64, device=v.device)
    else:
        grid = torch.arange(127, dtype=torch.uint8, device=v.device).view(torch.float8_e4m3fn).double()
    mid = (grid[1:] + grid[:-1]) / 2
    a = v.abs().contiguous()
    lo, hi = torch.searchsorted(mid, a), torch.searchsorted(mid, a, right=True)           # they differ on a tie only
    return torch.copysign(grid[torch.where(hi % 2 == 0, hi, lo)], v)


def _exact_mx(y, fmt):
    m, k = y.shape
    b = torch.nn.functional.pad(y, (0, padded(k) - k)).view(m, -1, 32)
    amax = b.abs().amax(2)
    e = torch.floor(torch.log2(amax)) - EMAX[fmt]
    e = torch.where(torch.exp2(e + EMAX[fmt]) > amax, e - 1, torch.where(torch.exp2(e + EMAX[fmt] + 1) <= amax, e + 1, e))
    e = torch.where(amax < 2.0 ** -126, torch.full_like(e, -127), e.clamp(-127, 127))
    c = _exact_round(b / torch.exp2(e)[..., None], fmt)
    if fmt == "fp8":
        return {"codes": c.view(m, -1), "scales": torch.exp2(e).view(m, -1, 4).transpose(0, 1)}
    return {"values": (c * torch.exp2(e)[..., None]).view(m, -1)[:, :k], "scales": torch.exp2(e).view(m, -1, 4).transpose(0, 1)}


def _exact_values(codes, scales, fmt):
    v = codes.int()
    if fmt == "fp4":
        v = torch.stack((v & 15, v >> 4), 2).flatten(1)
        sign, e, f = (v >> 3) & 1, (v >> 1) & 3, (v & 1).double() / 2
        bias = 1
    else:
        sign, e, f = v >> 7, (v >> 3) & 15, (v & 7).double() / 8
        bias = 7
    a = torch.where(e > 0, (1 + f) * torch.exp2((e - bias).double()), f * 2.0 ** (1 - bias))
    return torch.where(sign > 0, -a, a) * torch.exp2(scales.double() - 127).permute(1, 0, 2).flatten(1).repeat_interleave(32, 1)


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        h = s["x"].double()
        if s["residual"] is not None:
            h = h + s["residual"].double()
        y = h / torch.sqrt(h.square().sum(1, keepdim=True) / case["width"] + EPS) * s["gamma"].double()
        out = _exact_mx(y, case["out"]) if case["out"] in EMAX else {"y": y}
        if s["residual"] is not None:
            out["h"] = h
        return out
    if op == "quant":
        return _exact_mx(s["x"].double(), case["fmt"])
    if op == "gemm":
        c = torch.mm(_exact_values(s["a"], s["a_scales"], case["a"]), _exact_values(s["w"], s["w_scales"], "fp4").t().contiguous())
        if s["bias"] is not None:
            c = c + s["bias"].double()
        if case["act"] == "gelu":
            c = c * 0.5 * torch.special.erfc(-c / math.sqrt(2))
        elif case["act"] == "relu":
            c = torch.relu(c)
        return c if s["residual"] is None else c + s["residual"].double()
    p, d = case["pairs"], case["dim"]
    turn = torch.polar(torch.ones(case["tokens"], p, dtype=torch.float64, device="cuda"),
                       s["pos"].double()[s["axis"].long()].t().contiguous() * s["freq"])
    out = {}
    for name in ("q", "k"):
        if s[name] is None:
            continue
        x = s[name].double()
        first = torch.arange(p, device="cuda") * (1 if case["half"] else 2)
        second = first + (p if case["half"] else 1)
        z = torch.complex(x[..., first], x[..., second]) * turn.repeat(case["images"], 1)[:, None]
        out[name] = x.index_copy(2, first, z.real).index_copy(2, second, z.imag)
    return out


# ----------------------------------------------------------------------------------------------------------------- work
def _mx_bytes(m, k, fmt):
    return m * padded(k) * BYTES[fmt] + m * padded(k) / 32


def _mx_out_bytes(m, k, fmt):
    return _mx_bytes(m, k, fmt) if fmt == "fp8" else m * k * 2 + m * padded(k) / 32


def work(case):
    op = case["op"]
    if op == "norm":
        n = case["rows"] * case["width"]
        b = n * BYTES[case["x"]] + case["width"] * 4
        b += 0 if case["res"] == "none" else 2 * n * BYTES[case["res"]]
        b += _mx_out_bytes(case["rows"], case["width"], case["out"]) if case["out"] in EMAX else n * BYTES[case["out"]]
        return {"bytes": b, "flops": 5 * n}
    if op == "quant":
        n = case["rows"] * case["width"]
        return {"bytes": n * BYTES[case["x"]] + _mx_out_bytes(case["rows"], case["width"], case["fmt"]), "flops": 3 * n}
    if op == "gemm":
        m, n, k = case["rows"], case["cols"], case["width"]
        b = _mx_bytes(m, k, case["a"]) + _mx_bytes(n, k, "fp4") + m * n * BYTES[case["out"]] + (4 * n if case["bias"] else 0)
        b += 0 if case["res"] == "none" else m * n * BYTES[case["res"]]
        return {"bytes": b, "flops": 2 * m * n * k}
    n = case["tokens"] * case["images"] * (case["heads"] + case["kv"])
    return {"bytes": 2 * n * case["dim"] * BYTES[case["x"]] + 4 * case["axes"] * case["tokens"] + 12 * case["pairs"],
            "flops": 6 * n * case["pairs"]}
