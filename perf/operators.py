"""Cases for measuring the 4-bit operators and the query/key norm with rotation.

Five operators of a decoder layer whose linears run in microscaled 4-bit floating point
(MXFP4: blocks of 32 e2m1 values along K sharing one e8m0 power-of-two scale):

    quant      quant_mxfp4             an activation or a weight to 4 bits
    norm       add_rmsnorm_quant_mxfp4 residual add + RMSNorm + 4 bits
    silu       silu_mul_quant_mxfp4    silu(gate) * up + 4 bits
    mm         w4a4_mm                 the product of two 4-bit operands
    qk         qk_norm_rope            RMSNorm of each query/key head + position rotation

With `own` false, run() computes them with elementary torch operations; with `own` true it
makes the calls a user makes of int8_linear.  What an operator holds in 4 bits comes back
as the values it stands for (dequant_mxfp4).

The definitions, which exact() restates in 64 bits:
  block      amax = max|y| of 32 values; e = max(floor(log2 amax) - 2, -127);
             value = 2^e * RNE_e2m1(y / 2^e), saturated at 6 * 2^e.
  norm       h = x + residual; residual_out = round(h); r = float32(1 / sqrt(mean h^2 + eps));
             y = round(round(h * r) * weight), each in the activation's type (h, h * r and
             the product in float32).
  silu       y = round(float32(gate / (1 + exp(-gate)) * up)), round to the activation's type.
  mm         out = round(A @ B + bias).
  qk         n = x / sqrt(mean x^2 + eps) * weight for each head, then the first `rot`
             values rotated by the position's angles; one rounding at the end.
"""

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
ROPE_BASE = 1e6


# ------------------------------------------------------------------ cases

def listed():
    """Sizes of the two decoder shapes that the benchmark runs: hidden 2048, 16 query and 8
    key heads of 128, intermediate 6144; and hidden 4096, 32 and 8 heads, 14336."""
    return [
        # o_proj's input for one decode token: the smallest call, all latency
        {"name": "quant 1x2048", "op": "quant", "m": 1, "k": 2048, "dtype": "bf16"},
        # a prefill batch before o_proj of the larger model
        {"name": "quant 4096x4096", "op": "quant", "m": 4096, "k": 4096, "dtype": "bf16"},
        # decode batch, residual stream into the qkv linear
        {"name": "norm 17x2048", "op": "norm", "m": 17, "k": 2048, "dtype": "bf16"},
        # prefill batch of the larger model, fp16 activations, a ragged number of tokens
        {"name": "norm 2049x4096 fp16", "op": "norm", "m": 2049, "k": 4096, "dtype": "fp16"},
        # decode batch between gate_up and down of the larger model
        {"name": "silu 8x14336", "op": "silu", "m": 8, "k": 14336, "dtype": "bf16"},
        # prefill batch between gate_up and down
        {"name": "silu 4096x6144", "op": "silu", "m": 4096, "k": 6144, "dtype": "bf16"},
        # one token through qkv: streaming the weight
        {"name": "mm 1x4096x2048", "op": "mm", "m": 1, "n": 4096, "k": 2048, "dtype": "bf16", "bias": False},
        # a decode batch through down of the larger model: long K, few output tiles
        {"name": "mm 64x4096x14336", "op": "mm", "m": 64, "n": 4096, "k": 14336, "dtype": "bf16", "bias": True},
        # a short ragged prompt through the larger model's qkv, fp16
        {"name": "mm 333x6144x4096 fp16", "op": "mm", "m": 333, "n": 6144, "k": 4096, "dtype": "fp16", "bias": True},
        # a prefill batch through gate_up: the most arithmetic
        {"name": "mm 4096x12288x2048", "op": "mm", "m": 4096, "n": 12288, "k": 2048, "dtype": "bf16", "bias": False},
        # one decode token's heads
        {"name": "qk 1 token", "op": "qk", "m": 1, "heads": 16, "kv": 8, "dim": 128, "rot": 128,
         "pairs": False, "dtype": "bf16"},
        # a prefill batch of the larger model's heads
        {"name": "qk 4096 tokens", "op": "qk", "m": 4096, "heads": 32, "kv": 8, "dim": 128, "rot": 128,
         "pairs": False, "dtype": "bf16"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["quant", "norm", "silu", "mm", "mm", "qk"])
    case = {"op": op, "m": _log_int(rng, 1, 4096), "dtype": rng.choice(["bf16", "bf16", "fp16"])}
    if op == "qk":
        dim = rng.choice([64, 96, 128, 128, 256])
        kv = rng.choice([1, 2, 4, 8])
        case.update(heads=kv * rng.choice([1, 2, 3, 4]), kv=kv, dim=dim, rot=rng.choice([dim, dim, dim // 2]),
                    pairs=rng.choice([False, False, True]))
        return case
    case["k"] = 32 * _log_int(rng, 16, 448)
    if op == "mm":
        case.update(n=_log_int(rng, 256, 12288), bias=rng.choice([False, True]))
        while case["m"] * case["n"] * case["k"] > 4096 * 12288 * 2048:
            case["m"] = max(1, case["m"] // 2)
    elif case["m"] * case["k"] > 4096 * 6144:
        case["m"] = 4096 * 6144 // case["k"]
    return case


def work(case):
    m, t = case["m"], 2
    if case["op"] == "qk":
        d = (case["heads"] + case["kv"]) * case["dim"]
        # the rotation reads one row of angles a token (float32 cosines and sines)
        return {"bytes": 2 * t * m * d + 4 * m * case["rot"] + 8 * m + 2 * t * case["dim"], "flops": 8 * m * d}
    k = case["k"]
    if case["op"] == "quant":
        return {"bytes": 2 * t * m * k, "flops": 4 * m * k}
    if case["op"] == "norm":
        return {"bytes": 4 * t * m * k + t * k, "flops": 9 * m * k}
    if case["op"] == "silu":
        return {"bytes": 3 * t * m * k, "flops": 12 * m * k}
    n = case["n"]
    operands = (m + n) * (k // 2 + k // 32)
    return {"bytes": operands + t * m * n + (t * n if case["bias"] else 0), "flops": 2 * m * n * k}


# ------------------------------------------------------------------ inputs

def _randn(shape, g):
    return torch.randn(shape, generator=g, device=DEVICE)


def _activation(m, k, g, dtype):
    """Normal values whose channels have different sizes, as a residual stream's have, with
    a few rows of zeros (padding tokens) in a batch that has room for them."""
    x = _randn((m, k), g) * torch.exp(0.5 * _randn((1, k), g))
    if m >= 64:
        x[m // 3] = 0
    return x.to(dtype)


def _tiled_scales(e):
    """Scale bytes [rows, blocks] in the layout of the product's operands: tiles of 128 rows
    x 4 blocks, 512 bytes each, row r's four bytes at (r % 32) * 16 + (r // 32) * 4; the
    tiles of one 128-row group in order of K; zero where a tile passes the matrix's end."""
    rows, blocks = e.shape
    rt, kt = -(-rows // 128), -(-blocks // 4)
    full = torch.zeros((rt * 128, kt * 4), dtype=torch.uint8, device=e.device)
    full[:rows, :blocks] = e
    return full.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(rt, kt, 512).contiguous()


def _operand(rows, k, g, scale):
    """A 4-bit operand as a user holds it: packed codes [rows, k/2] and tiled scale bytes."""
    codes, e = _codes(_randn((rows, k), g) * torch.exp(0.5 * _randn((1, k), g)) * scale)
    codes = codes.view(rows, k).to(torch.uint8)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), _tiled_scales((e + 127).to(torch.uint8))


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, m = TYPES[case["dtype"]], case["m"]
    state = {"case": case, "dtype": dtype}
    if case["op"] == "quant":
        state["x"] = _activation(m, case["k"], g, dtype)
    elif case["op"] == "norm":
        state["x"] = _activation(m, case["k"], g, dtype)
        state["residual"] = (2 * _randn((m, case["k"]), g)).to(dtype)
        state["weight"] = (1 + 0.1 * _randn((case["k"],), g)).to(dtype)
    elif case["op"] == "silu":
        state["gate_up"] = _activation(m, 2 * case["k"], g, dtype)
    elif case["op"] == "mm":
        state["a"], state["sa"] = _operand(m, case["k"], g, 1.0)
        state["b"], state["sb"] = _operand(case["n"], case["k"], g, 0.02)
        state["bias"] = (0.01 * _randn((case["n"],), g)).to(dtype) if case["bias"] else None
    else:
        d, rot = case["dim"], case["rot"]
        state["qkv"] = _activation(m, (case["heads"] + 2 * case["kv"]) * d, g, dtype)
        state["wq"], state["wk"] = ((1 + 0.1 * _randn((d,), g)).to(dtype) for _ in range(2))
        length = 8192
        state["positions"] = torch.randint(0, length, (m,), generator=g, device=DEVICE)
        freq = ROPE_BASE ** (-torch.arange(0, rot, 2, device=DEVICE, dtype=torch.float64) / rot)
        angle = torch.arange(length, device=DEVICE, dtype=torch.float64)[:, None] * freq
        state["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
    return state


# ------------------------------------------------------------------ the operators

def run(s):
    return {"quant": _quant, "norm": _norm, "silu": _silu, "mm": _mm, "qk": _qk}[s["case"]["op"]](s)


def _quant(s):
    if own:
        from int8_linear import mxfp4
        return mxfp4.dequant_mxfp4(*mxfp4.quant_mxfp4(s["x"]), s["dtype"])
    return _values(s["x"].float()).to(s["dtype"])


def _norm(s):
    if own:
        from int8_linear import mxfp4
        q, e, out = mxfp4.add_rmsnorm_quant_mxfp4(s["x"], s["residual"], s["weight"], EPS)
        return mxfp4.dequant_mxfp4(q, e, s["dtype"]), out
    h = s["x"].float() + s["residual"].float()
    # the mean in 64 bits: a rounding of r away from its float32 value moves values next to
    # a border of the 4-bit type across it
    r = (1 / torch.sqrt(h.double().square().mean(1, keepdim=True) + EPS)).float()
    y = ((h * r).to(s["dtype"]).float() * s["weight"].float()).to(s["dtype"])
    return _values(y.float()).to(s["dtype"]), h.to(s["dtype"])


def _silu(s):
    if own:
        from int8_linear import mxfp4
        return mxfp4.dequant_mxfp4(*mxfp4.silu_mul_quant_mxfp4(s["gate_up"]), s["dtype"])
    # in 64 bits, rounded to 32: values next to a border, as above
    gate, up = s["gate_up"].double().chunk(2, 1)
    y = (gate / (1 + torch.exp(-gate)) * up).float().to(s["dtype"])
    return _values(y.float()).to(s["dtype"])


def _mm(s):
    if own:
        from int8_linear import mxfp4
        return mxfp4.w4a4_mm(s["a"], s["b"].t(), s["sa"], s["sb"], s["dtype"], s["bias"])
    out = _unpack(s["a"], s["sa"]) @ _unpack(s["b"], s["sb"]).t()
    return (out if s["bias"] is None else out + s["bias"].float()).to(s["dtype"])


def _qk(s):
    c = s["case"]
    if own:
        from int8_linear.qk_norm import qk_norm_rope
        return qk_norm_rope(s["qkv"], s["wq"], s["wk"], EPS, s["positions"], s["cos_sin"],
                            c["heads"], c["kv"], interleaved=c["pairs"])
    heads = s["qkv"].view(c["m"], -1, c["dim"]).float()
    angles = s["cos_sin"][s["positions"]][:, None]
    split = (c["heads"], c["heads"] + c["kv"])
    return tuple(_norm_rotate(x, w.float(), angles, c["rot"], c["pairs"]).to(s["dtype"])
                 for x, w in ((heads[:, :split[0]], s["wq"]), (heads[:, split[0]:split[1]], s["wk"])))


# ------------------------------------------------------------------ plain forms

def _codes(x):
    """e2m1 codes [rows, blocks, 32] (int64) of float32 x, and the block exponents."""
    b = x.view(x.shape[0], -1, 32)
    e = (torch.frexp(b.abs().amax(2)).exponent - 3).clamp(min=-127)
    a = b * ((127 - e) << 23).view(torch.float32)[..., None]
    mag = a.abs()
    # halves of a step go to the even code
    code = ((mag > 0.25).long() + (mag >= 0.75) + (mag > 1.25) + (mag >= 1.75) + (mag > 2.5) + (mag >= 3.5)
            + (mag > 5))
    return code + 8 * (a < 0), e


_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)


def _values(x):
    """x after a trip through 4 bits, in float32."""
    codes, e = _codes(x)
    v = torch.tensor(_E2M1, device=x.device)[codes]
    return (v * torch.exp2(e.float())[..., None]).view(x.shape)


def _unpack(q, s):
    """Packed codes and tiled scales to float32 values [rows, k]."""
    rows, k = q.shape[0], 2 * q.shape[1]
    codes = torch.stack([q & 15, q >> 4], 2).view(rows, k // 32, 32).long()
    rt, kt, _ = s.shape
    e = s.view(rt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:rows, :k // 32]
    v = torch.tensor(_E2M1, device=q.device)[codes]
    return (v * torch.exp2(e.float() - 127)[..., None]).view(rows, k)


def _norm_rotate(x, w, angles, rot, pairs):
    n = x * torch.rsqrt(x.square().mean(2, keepdim=True) + EPS) * w
    cos, sin = angles[..., :rot // 2], angles[..., rot // 2:]
    r = n[..., :rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if pairs else (r[..., :rot // 2], r[..., rot // 2:])
    turned = (a * cos - b * sin, b * cos + a * sin)
    turned = torch.stack(turned, -1).flatten(-2) if pairs else torch.cat(turned, -1)
    return torch.cat([turned, n[..., rot:]], -1)


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_values(y):
    """Block rounding of float64 y by the borders between neighbouring 4-bit values."""
    grid = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=y.device)
    middle = (grid[1:] + grid[:-1]) / 2
    b = y.view(-1, 32)
    top = b.abs().amax(1, keepdim=True)
    powers = torch.tensor([2.0 ** i for i in range(-160, 160)], dtype=torch.float64, device=y.device)
    e = torch.searchsorted(powers, top, right=True) - 1 - 160  # the largest power of two not above it
    unit = powers[(e - 2).clamp(min=-127) + 160]
    mag = (b / unit).abs()
    low = torch.searchsorted(middle, mag)               # a border itself counts as below it
    high = torch.searchsorted(middle, mag, right=True)  # ... and here as above
    index = torch.where(low % 2 == 0, low, high)        # at a border: the even one of the two
    return (torch.sign(b) * grid[index] * unit).view(y.shape)


def _exact_operand(q, s):
    rows, half = q.shape
    r = torch.arange(rows, device=q.device)[:, None]
    j = torch.arange(2 * half // 32, device=q.device)[None]
    byte = s[r // 128, j // 4, (r % 32) * 16 + (r % 128) // 32 * 4 + j % 4].double()
    code = torch.empty((rows, 2 * half), dtype=torch.int32, device=q.device)
    code[:, 0::2], code[:, 1::2] = (q % 16).int(), (q // 16).int()
    exponent, mantissa = code // 2 % 4, code % 2
    mag = torch.where(exponent == 0, 0.5 * mantissa, (1 + 0.5 * mantissa) * torch.exp2(exponent.double() - 1))
    return torch.where(code >= 8, -mag, mag) * torch.exp2(byte - 127).repeat_interleave(32, 1)


def exact(case, seed):
    s = prepare(case, seed)
    dtype = s["dtype"]
    if case["op"] == "quant":
        return _exact_values(s["x"].double())
    if case["op"] == "norm":
        h = s["x"].double() + s["residual"].double()
        h32 = h.float().double()  # the sum is held in float32
        rms = torch.sqrt((h32 * h32).sum(1, keepdim=True) / case["k"] + EPS)
        r = torch.reciprocal(rms).float().double()
        y = (h32 * r).float().to(dtype).double() * s["weight"].double()
        return _exact_values(y.float().to(dtype).double()), h
    if case["op"] == "silu":
        gate, up = s["gate_up"][:, :case["k"]].double(), s["gate_up"][:, case["k"]:].double()
        return _exact_values((gate * up * torch.sigmoid(gate)).float().to(dtype).double())
    if case["op"] == "mm":
        out = torch.einsum("mk,nk->mn", _exact_operand(s["a"], s["sa"]), _exact_operand(s["b"], s["sb"]))
        return out if s["bias"] is None else out + s["bias"].double()[None]
    d, rot, half = case["dim"], case["rot"], case["rot"] // 2
    table = s["cos_sin"].double()[s["positions"]]
    cos, sin = table[:, None, :half], table[:, None, half:]
    first = torch.arange(half, device=DEVICE) * (2 if case["pairs"] else 1)
    second = first + (1 if case["pairs"] else half)
    outs, begin = [], 0
    for heads, w in ((case["heads"], s["wq"]), (case["kv"], s["wk"])):
        x = s["qkv"][:, begin:begin + heads * d].double().reshape(case["m"], heads, d)
        begin += heads * d
        n = x / torch.sqrt((x * x).sum(2, keepdim=True) / d + EPS) * w.double()
        y = n.clone()
        y[..., first] = n[..., first] * cos - n[..., second] * sin
        y[..., second] = n[..., first] * sin + n[..., second] * cos
        outs.append(y)
    return tuple(outs)
