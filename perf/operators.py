"""The microscaled (block-scaled floating point) operators: what they compute, in plain torch operations, and their calls.

Three formats hold a matrix as codes and one scale per block of neighbouring columns of a row:

  nvfp4   e2m1 codes (4 bits), blocks of 16, e4m3 scales, one fp32 scale per tensor: x = code * scale * tensor scale
  mxfp4   e2m1 codes (4 bits), blocks of 32, power-of-two scales (e8m0)
  mxfp8   e4m3 codes (8 bits), blocks of 32, power-of-two scales (e8m0)

Codes are rows of K_pad = K rounded up to 128 columns (zero past K), 4-bit codes two to a byte with the even column in the low half.
Scales are bytes in tiles of 128 rows and 4 blocks: byte (row % 32) * 16 + (row / 32 % 4) * 4 + block % 4 of tile (row / 128, block / 4);
rows past the last one are zero.

Operators: "round_trip" quantises and reads back, "linear" quantises activations and multiplies them with a 4-bit weight, "product"
multiplies two matrices that are in these formats already, "norm" adds a residual, takes the root-mean-square norm and writes it as mxfp8.
"""
import torch

own = False

BLOCK = {"nvfp4": 16, "mxfp4": 32, "mxfp8": 32}
DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
EPS = 1e-6


def listed():
    return [
        # one token through a block's pre-norm: latency alone
        dict(name="norm_1_token", op="norm", m=1, k=6144, dtype="bf16", residual=True),
        # the pre-norm of a block at 1024 px (4096 image and 256 text tokens)
        dict(name="norm_block", op="norm", m=4352, k=6144, dtype="bf16", residual=True),
        # odd width: rows that start at no 16-byte boundary, a last block that is not full
        dict(name="norm_odd", op="norm", m=1027, k=1111, dtype="fp16", residual=False),
        # what 4 bits make of a block's activations
        dict(name="round_trip_nvfp4", op="round_trip", m=4352, k=6144, dtype="bf16", fmt="nvfp4", cut=0),
        # odd sizes, fp32, rows cut out of wider ones
        dict(name="round_trip_mxfp4_odd", op="round_trip", m=777, k=1001, dtype="fp32", fmt="mxfp4", cut=23),
        # one token through ff.up: bound by the weight's bytes
        dict(name="linear_nvfp4_1_token", op="linear", m=1, n=16384, k=6144, dtype="bf16", fmt="nvfp4", bias=True),
        # ff.down for 16 tokens, 8-bit activations on a 4-bit weight
        dict(name="linear_w4a8_16_tokens", op="linear", m=16, n=6144, k=16384, dtype="bf16", fmt="mxfp8", bias=True),
        # nothing is a multiple of a tile
        dict(name="linear_mxfp4_odd", op="linear", m=301, n=1537, k=1030, dtype="fp32", fmt="mxfp4", bias=True),
        # ff.up of a block at 1024 px
        dict(name="linear_nvfp4_block", op="linear", m=4352, n=16384, k=6144, dtype="bf16", fmt="nvfp4", bias=True),
        # a short prompt's keys from activations that are in the format already
        dict(name="product_mxfp4_64_tokens", op="product", m=64, n=1536, k=6144, dtype="fp32", fmt="mxfp4", bias=False),
        # the norm's output into the query projection
        dict(name="product_w4a8_block", op="product", m=4352, n=6144, k=6144, dtype="bf16", fmt="mxfp8", bias=False),
        # ff.up for four images at once
        dict(name="product_nvfp4_4_images", op="product", m=17408, n=16384, k=6144, dtype="bf16", fmt="nvfp4", bias=True),
    ]


def draw(rng):
    def size(lo, hi):
        v = int(round(lo * (hi / lo) ** rng.random()))
        return v if rng.random() < 0.5 else max(lo, v // 16 * 16)

    op = rng.choice(["norm", "round_trip", "linear", "linear", "product", "product"])
    case = dict(op=op, m=size(1, 8192), k=size(64, 16384), dtype=rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if op == "norm":
        case.update(residual=rng.random() < 0.7)
    elif op == "round_trip":
        case.update(fmt=rng.choice(["nvfp4", "mxfp4", "mxfp8"]), cut=rng.choice([0, 0, 8, 23]))
    else:
        case.update(n=size(64, 16384), fmt=rng.choice(["nvfp4", "mxfp4", "mxfp8"]), bias=rng.random() < 0.5)
    most = work(listed()[-1])
    while work(case)["flops"] > most["flops"] or work(case)["bytes"] > most["bytes"]:
        case["m"] = case["m"] * 2 // 3
    return case


def work(case):
    m, k, s = case["m"], case["k"], SIZE[case["dtype"]]
    coded = {f: (1 if f == "mxfp8" else 0.5) + 1 / b for f, b in BLOCK.items()}
    if case["op"] == "norm":
        return {"bytes": m * k * (s * (3 if case["residual"] else 1) + coded["mxfp8"]) + s * k, "flops": 6 * m * k}
    if case["op"] == "round_trip":
        return {"bytes": 2 * m * k * s, "flops": 4 * m * k}
    n, fmt = case["n"], case["fmt"]
    a = m * k * (s if case["op"] == "linear" else coded[fmt])
    return {"bytes": a + n * k * coded[_weight(fmt)] + m * n * s + 2 * n * case["bias"], "flops": 2 * m * n * k}


def _weight(fmt):
    """The weight's format beside activations in `fmt`: 8-bit activations take a 4-bit weight with scales of the same kind."""
    return "mxfp4" if fmt == "mxfp8" else fmt


# ---------------------------------------------------------------- plain forms


def _padded(k):
    return -(-k // 128) * 128


def _two(e):
    """2^e in 64 bits, from its bits."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _scale(amax, fmt, tensor_scale):
    """A block's scale from its largest magnitude, as a value: for the mx formats 2^(floor(log2 amax) - the exponent of the largest
    code), for nvfp4 e4m3(amax / (6 * tensor scale)) with ties to even."""
    if fmt != "nvfp4":
        e = torch.frexp(amax)[1] - 1 - (2 if fmt == "mxfp4" else 8)
        e = torch.where(amax > 0, e, -127).clamp(-127, 127)
        return _two(e).to(amax.dtype)
    t = (amax / (6 * tensor_scale.to(amax.dtype))).clamp(max=448)
    step = _two((torch.frexp(t)[1] - 1).clamp(min=-6) - 3).to(t.dtype)
    return torch.round(t / step) * step


def _e2m1(q):
    """The index 0..7 of the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6; halfway goes to the even index."""
    q = q.abs()
    return (q > 0.25).byte() + (q >= 0.75).byte() + (q > 1.25).byte() + (q >= 1.75).byte() + (q > 2.5).byte() + (q >= 3.5).byte() + (q > 5).byte()


def _quantize(x, fmt, tensor_scale, wide=torch.float64):
    """x [M, K] as (codes, scale values [M, blocks]); in 64 bits, so that no value next to a border goes to its wrong side."""
    m, k = x.shape
    b = BLOCK[fmt]
    x = torch.nn.functional.pad(x.to(wide), (0, _padded(k) - k)).view(m, -1, b)
    scale = _scale(x.abs().amax(-1), fmt, tensor_scale)
    unit = scale if fmt != "nvfp4" else scale * tensor_scale.to(wide)
    q = x / torch.where(unit > 0, unit, 1.0)[..., None]
    q = torch.where(unit[..., None] > 0, q, 0.0).view(m, -1)
    if fmt == "mxfp8":
        return _e4m3(q).to(torch.float8_e4m3fn), scale
    c = _e2m1(q) | (torch.signbit(q).byte() << 3)
    return c[:, 0::2] | (c[:, 1::2] << 4), scale


def _e4m3(q):
    """The nearest e4m3 value, halfway to the even one, at most 448 in magnitude."""
    step = _two((torch.frexp(q)[1] - 1).clamp(min=-6) - 3).to(q.dtype)
    return (torch.round(q / step) * step).clamp(-448, 448)


def _tiled(scale, fmt):
    """Scale values [M, blocks] as bytes in the tile order."""
    if fmt == "nvfp4":
        s = scale.float().to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        s = (torch.frexp(scale)[1] - 1 + 127).byte()
    m, c = s.shape
    s = torch.nn.functional.pad(s, (0, 0, 0, _padded(m) - m))
    return s.view(-1, 4, 32, c // 4, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def _untiled(tiled, m, k, fmt):
    """Bytes in the tile order as scale values [M, blocks] in 32 bits."""
    c = _padded(k) // BLOCK[fmt]
    s = tiled.view(-1, c // 4, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, c)[:m].contiguous()
    if fmt == "nvfp4":
        return s.view(torch.float8_e4m3fn).float()
    return _two(s.int() - 127).float()


def _values(codes, scale, fmt, tensor_scale):
    """Codes and scale values [M, blocks] as the values [M, K_pad] that they stand for, in 32 bits."""
    if fmt == "mxfp8":
        v = codes.float()
    else:
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], device=codes.device)
        v = table[torch.stack((codes & 15, codes >> 4), -1).view(codes.shape[0], -1).int()]
    unit = scale.float() if fmt != "nvfp4" else scale.float() * tensor_scale
    return (v.view(v.shape[0], -1, BLOCK[fmt]) * unit[..., None]).view(v.shape[0], -1)


def _product(a, w, bias, dtype):
    y = a @ w.t()
    return (y if bias is None else y + bias.float()).to(dtype)


# ---------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda")

    def activations(m, k, cut=0):
        """N(0, 1) with one column in a hundred 20 times as large: the outlier channels of a transformer's activations."""
        far = torch.where(torch.rand(k + cut, generator=g, device="cuda") < 0.01, 20.0, 1.0)
        return (normal(m, k + cut) * far).to(DTYPE[case["dtype"]])[:, :k]

    m, k = case["m"], case["k"]
    state = dict(case)
    state["dtype"] = DTYPE[case["dtype"]]
    if case["op"] == "norm":
        state["x"] = activations(m, k)
        state["residual"] = activations(m, k) if case["residual"] else None
        state["weight"] = (1 + 0.1 * normal(k)).to(state["dtype"])
        return state
    fmt = case["fmt"]
    # a calibrated tensor scale: the largest activation lands on the largest code and scale
    state["act_scale"] = torch.tensor([90.0 / (6 * 448)], device="cuda") if fmt == "nvfp4" else None
    x = activations(m, k, case.get("cut", 0))
    if case["op"] == "round_trip":
        state["x"] = x
        return state
    w, wf = 0.02 * normal(case["n"], k), _weight(fmt)
    state["w_scale"] = (w.abs().amax() / (6 * 448)).view(1) if wf == "nvfp4" else None
    codes, scale = _quantize(w, wf, state["w_scale"], torch.float32)
    state["w_codes"], state["w_scales"] = codes, _tiled(scale, wf)
    del w
    state["bias"] = (0.01 * normal(case["n"])).to(torch.bfloat16) if case["bias"] else None
    if case["op"] == "linear":
        state["x"] = x
    else:
        codes, scale = _quantize(x, fmt, state["act_scale"], torch.float32)
        state["a_codes"], state["a_scales"] = codes, _tiled(scale, fmt)
    return state


# ---------------------------------------------------------------- one pass


def run(s):
    if own:
        return _run_own(s)
    op, m, k = s["op"], s["m"], s["k"]
    if op == "norm":
        h = s["x"] if s["residual"] is None else (s["x"].float() + s["residual"].float()).to(s["dtype"])
        v = h.float()
        v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
        codes, scale = _quantize(v, "mxfp8", None, torch.float32)
        out = {"codes": codes, "scales": _tiled(scale, "mxfp8").view(torch.float8_e8m0fnu)}
        return out if s["residual"] is None else dict(out, sum=h)
    fmt, wf = s["fmt"], _weight(s["fmt"])
    if op == "round_trip":
        codes, scale = _quantize(s["x"], fmt, s["act_scale"])
        return _values(codes, scale, fmt, s["act_scale"])[:, :k].to(s["dtype"])
    w = _values(s["w_codes"], _untiled(s["w_scales"], s["n"], k, wf), wf, s["w_scale"])
    if op == "linear":
        codes, scale = _quantize(s["x"], fmt, s["act_scale"])
    else:
        codes, scale = s["a_codes"], _untiled(s["a_scales"], m, k, fmt)
    return _product(_values(codes, scale, fmt, s["act_scale"]), w, s["bias"], s["dtype"])


def _run_own(s):
    from krea2_svdquant_b200 import microscale as ms

    op = s["op"]
    if op == "norm":
        t, h = ms.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        out = {"codes": t.codes, "scales": t.scales.view(torch.float8_e8m0fnu)}
        return out if s["residual"] is None else dict(out, sum=h)
    fmt = s["fmt"]
    if op == "round_trip":
        return ms.dequantize(ms.quantize(s["x"], fmt, tensor_scale=s["act_scale"]), s["dtype"])
    w = ms.MicroTensor(s["w_codes"], s["w_scales"], _weight(fmt), (s["n"], s["k"]), s["w_scale"])
    if op == "linear":
        return ms.linear(s["x"], w, s["bias"], act=fmt, act_scale=s["act_scale"])
    a = ms.MicroTensor(s["a_codes"], s["a_scales"], fmt, (s["m"], s["k"]), s["act_scale"])
    return ms.matmul(a, w, s["bias"], out_dtype=s["dtype"])


# ---------------------------------------------------------------- the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    op, m, k = s["op"], s["m"], s["k"]
    d = torch.float64

    def power(v):  # the exponent of the largest power of two that is not above v > 0
        return torch.frexp(v)[1] - 1

    def two(e):
        return torch.exp2(e.to(d))

    def nearest(v, bits, low, top):  # v rounded, halfway to even, to `bits` fraction bits above 2^low, at most `top`
        u = two(torch.clamp(power(v), min=low) - bits)
        return torch.clamp(torch.round(v / u) * u, -top, top)

    def blocks_of(v, b):
        out = torch.zeros(v.shape[0], -(-k // 128) * 128, dtype=d, device=v.device)
        out[:, :k] = v
        return out.view(v.shape[0], -1, b)

    def coded(v, fmt):
        """v [M, K] as (what its codes say, its blocks' scales)."""
        v = blocks_of(v, 16 if fmt == "nvfp4" else 32)
        top = v.abs().max(-1).values
        if fmt == "nvfp4":
            scale = nearest(top / (6 * s["act_scale"].to(d)), 3, -6, 448)
            unit = (scale * s["act_scale"].to(d))[..., None]
        else:
            scale = two(torch.clamp(torch.where(top > 0, power(top) - (8 if fmt == "mxfp8" else 2), -127), -127, 127))
            unit = scale[..., None]
        q = torch.where(unit != 0, v / unit, torch.zeros_like(v))
        return (nearest(q, 3, -6, 448) if fmt == "mxfp8" else nearest(q, 1, 0, 6)), scale, unit

    def held(codes, scales, rows, fmt, tensor_scale):
        """The values that codes and tiled scales stand for."""
        b = 16 if fmt == "nvfp4" else 32
        r = torch.arange(rows, device=codes.device)[:, None]
        c = torch.arange(-(-k // 128) * 128 // b, device=codes.device)[None, :]
        at = ((r // 128) * (c.shape[1] // 4) + c // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + c % 4
        s8 = scales[at]
        unit = s8.view(torch.float8_e4m3fn).to(d) * tensor_scale.to(d) if fmt == "nvfp4" else two(s8.int() - 127)
        if fmt == "mxfp8":
            v = codes.to(d)
        else:
            v = torch.empty(rows, codes.shape[1] * 2, dtype=d, device=codes.device)
            v[:, 0::2], v[:, 1::2] = _e2m1_exact(codes % 16), _e2m1_exact(codes // 16)
        return (v.view(rows, -1, b) * unit[..., None]).flatten(1)[:, :k]

    if op == "norm":
        x = s["x"].to(d)
        total = x if s["residual"] is None else x + s["residual"].to(d)
        h = total.to(s["dtype"]).to(d)  # the norm is that of the sum as it is stored
        y = h / torch.sqrt((h * h).sum(-1, keepdim=True) / k + EPS) * s["weight"].to(d)
        q, scale, _ = coded(y, "mxfp8")
        rows, blocks = scale.shape
        full = torch.full((-(-rows // 128) * 128, blocks), 2.0 ** -127, dtype=d, device=x.device)
        full[:rows] = scale
        tiles = torch.stack(full.view(-1, 128, blocks).split(32, 1), 2)  # [tile, row % 32, row / 32, block]
        tiles = torch.stack(tiles.split(4, -1), 1).reshape(-1)
        out = {"codes": q.flatten(1), "scales": tiles}
        return out if s["residual"] is None else dict(out, sum=total)
    fmt = s["fmt"]
    if op == "round_trip":
        q, _, unit = coded(s["x"].to(d), fmt)
        return (q * unit).flatten(1)[:, :k]
    if op == "linear":
        q, _, unit = coded(s["x"].to(d), fmt)
        a = (q * unit).flatten(1)[:, :k]
    else:
        a = held(s["a_codes"], s["a_scales"], m, fmt, s["act_scale"])
    y = a @ held(s["w_codes"], s["w_scales"], s["n"], _weight(fmt), s["w_scale"]).t()
    return y if s["bias"] is None else y + s["bias"].to(d)


def _e2m1_exact(c):
    """The value of a 4-bit code: a sign, two exponent bits (bias 1) and one fraction bit."""
    e, f = (c // 2 % 4).double(), (c % 2).double()
    v = torch.where(e > 0, torch.exp2(e - 1) * (1 + f / 2), f / 2)
    return torch.where(c >= 8, -v, v)
