"""Block-scaled formats on the GPU: quantisation, reading back, products and the norm, against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FORMATS = ("nvfp4", "mxfp4", "mxfp8")
PRODUCTS = (("nvfp4", "nvfp4"), ("mxfp4", "mxfp4"), ("mxfp8", "mxfp4"))


def ms():
    from krea2_svdquant_b200 import microscale
    return microscale


def no_device_error():
    from krea2_svdquant_b200 import _lib
    assert _lib.device_error() == 0


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def data(m, k, dtype=torch.float32, seed=0, cut=0, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(m, k + cut, generator=g) * scale
    x[:, ::37] *= 20
    return x.to(dtype).cuda()[:, :k]


def code_bytes(t) -> np.ndarray:
    return t.codes.view(torch.uint8).cpu().numpy()


def check_quantized(t, x, fmt, g=1.0):
    """Codes, scales and padding of t against the definition, bit for bit; returns the oracle's values."""
    m, k = x.shape
    codes, byte = O.quantize(f64(x), fmt, g)
    scales = t.scales.cpu().numpy()
    at = O.scale_index(m, byte.shape[1])
    np.testing.assert_array_equal(scales[at], byte)
    rest = np.ones(scales.size, bool)
    rest[at.ravel()] = False
    assert not scales[rest].any(), "scales of rows past the last one"
    np.testing.assert_array_equal(O.unpack(code_bytes(t), fmt), codes)
    return O.values(codes, byte, fmt, g)[:, :k]


def operand_values(t) -> np.ndarray:
    """The values [rows, K] of a MicroTensor, decoded by the oracle."""
    k = t.shape[-1]
    rows = t.codes.shape[0]
    byte = t.scales.cpu().numpy()[O.scale_index(rows, O.k_pad(k) // O.BLOCK[t.fmt])]
    g = 1.0 if t.tensor_scale is None else float(t.tensor_scale)
    return O.values(O.unpack(code_bytes(t), t.fmt), byte, t.fmt, g)[:, :k]


def check_product(y, a, w, bias, dtype):
    """y against A W^T + bias in 64 bits.  The tensor core adds in fp32 and may truncate, so each of the
    K additions loses at most 2^-23 of the sum of magnitudes; alpha, bias and the output round by half a
    step each.  Over all elements the errors do not line up: 1e-5 of the norm plus the output's rounding."""
    s = np.abs(a) @ np.abs(w).T
    ref = a @ w.T
    if bias is not None:
        ref, s = ref + f64(bias), s + np.abs(f64(bias))
    u = torch.finfo(dtype).eps / 2
    tiny = float(torch.finfo(dtype).smallest_normal) * torch.finfo(dtype).eps
    got = f64(y)
    bound = a.shape[1] * 2.0 ** -23 * s + 3 * 2.0 ** -24 * s + u * (np.abs(ref) + a.shape[1] * 2.0 ** -23 * s) + tiny
    assert got.shape == ref.shape
    assert (np.abs(got - ref) <= bound).all(), float((np.abs(got - ref) - bound).max())
    rel = np.linalg.norm(got - ref) / max(np.linalg.norm(ref), 1e-300)
    assert rel <= 1e-5 + u, rel


# ------------------------------------------------------------------ quantisation
@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("m,k,cut", [(1, 1, 0), (1, 6144, 0), (127, 15, 0), (128, 16, 0), (129, 17, 5), (3, 129, 0),
                                     (200, 1000, 24), (65, 333, 3)])
def test_quantize_is_the_definition(fmt, dtype, m, k, cut):
    x = data(m, k, DTYPES[dtype], seed=m + k, cut=cut)
    t = ms().quantize(x, fmt)
    ref = check_quantized(t, x, fmt)
    for out in DTYPES.values():  # values have at most 8 significant bits: exact in every type that has their range
        got = f64(ms().dequantize(t, out))
        half = 0.0 if out != torch.float16 else torch.finfo(out).smallest_normal * torch.finfo(out).eps / 2
        assert (np.abs(got - ref) <= half).all()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("g", [1.0, 0.25, 0.0371, 3.1415927e-20, 7.3e-35, 1.7e20, 0.3333333433])
def test_nvfp4_tensor_scale(dtype, g):
    g = np.float32(g)
    s = float(np.clip(g, 1e-4, 1e3)) if dtype == "fp16" else float(g)
    x = data(33, 640, DTYPES[dtype], seed=5, scale=s * 3)
    scale = torch.tensor([g], device="cuda")
    check_quantized(ms().quantize(x, "nvfp4", tensor_scale=scale), x, "nvfp4", float(g))


@pytest.mark.parametrize("fmt", FORMATS)
def test_borders_go_to_the_even_code(fmt):
    """Every midpoint between two codes, its neighbours and the codes themselves, in blocks whose scale
    is fixed by a largest element, times every scale that a byte can hold."""
    table = O.E4M3[:127] if fmt == "mxfp8" else O.E2M1[:8]
    mid = (table[1:] + table[:-1]) / 2
    pts = np.concatenate([mid, np.nextafter(mid.astype(np.float32), np.float32(0)), np.nextafter(mid.astype(np.float32), np.float32(9e9)), table])
    pts = np.concatenate([pts, -pts]).astype(np.float64)
    b = O.BLOCK[fmt]
    rows = -(-pts.size // (b - 1))
    blocks = np.zeros((rows, b))
    blocks[:, 0] = table[-1]
    blocks[:, 1:].flat[:pts.size] = pts
    sf = O.E4M3[1:127] if fmt == "nvfp4" else np.ldexp(1.0, np.arange(-110, 111, 5))
    x = (sf[:, None, None] * blocks[None]).astype(np.float32).reshape(len(sf), -1)
    xt = torch.from_numpy(x).cuda()
    check_quantized(ms().quantize(xt, fmt), xt, fmt)


def test_borders_with_a_tensor_scale_of_24_bits():
    """x next to border * scale * g, where sf * g is not an fp32 value: the code is that of the exact quotient."""
    rng = np.random.default_rng(3)
    g = np.float32(0.7853981633974483)
    sf = O.E4M3[rng.integers(9, 127, (400, 1))]
    mid = rng.choice((O.E2M1[1:8] + O.E2M1[:7]) / 2, (400, 16)) * rng.choice([-1, 1], (400, 16))
    x = (sf * np.float64(g) * mid).astype(np.float32)
    x = np.where(rng.random(x.shape) < 0.3, np.nextafter(x, np.float32(0)), x)
    x[:, 0] = (sf[:, 0] * np.float64(g) * 6).astype(np.float32)
    xt = torch.from_numpy(x.reshape(50, 128)).cuda()
    check_quantized(ms().quantize(xt, "nvfp4", tensor_scale=torch.tensor([g], device="cuda")), xt, "nvfp4", float(g))


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("g", [1.0, 0.75, 90 / 2688, 15 / 448, 13.25 / 2688, 1 / 3, 0.1, 0.0371, 1 + 2.0 ** -23, 1 + 2.0 ** -9,
                               0.25 * (1 + 2.0 ** -17), 0.25 * (1 - 2.0 ** -19), 8 / 7, 1 / 7 + 2.0 ** -26, 4 / 5 - 2.0 ** -22])
def test_borders_of_16_bit_inputs(dtype, g):
    """The 16-bit numbers nearest to every border times every scale times g, and their neighbours: tensor scales
    that put none, one, some or all of them on their borders, exactly or nearly."""
    t, g = DTYPES[dtype], np.float32(g)
    sf = O.E4M3[16:120]
    mid = (O.E2M1[1:8] + O.E2M1[:7]) / 2
    unit = (sf * np.float64(g))[:, None]
    x = torch.from_numpy(unit * mid).to(t)
    near = x.view(torch.int16)
    rows = torch.cat([x, (near + 1).view(t), (near - 1).view(t)], 1)  # 21 a scale, in two blocks of 16
    rows = torch.cat([rows[:, :11], rows[:, 11:], -rows[:, :8]], 1)[:, :30]
    top = torch.from_numpy(unit * 6).to(t)
    blocks = torch.cat([top, rows[:, :15], top, rows[:, 15:]], 1).contiguous()
    check_quantized(ms().quantize(blocks.cuda(), "nvfp4", tensor_scale=torch.tensor([g], device="cuda")), blocks,
                    "nvfp4", float(g))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_extreme_values(fmt, dtype):
    t = DTYPES[dtype]
    x = torch.zeros(8, 256, dtype=t)
    big, small = torch.finfo(t).max, torch.finfo(t).smallest_normal
    x[0, :32] = big
    x[0, 32:64] = -big
    x[1] = torch.linspace(-1, 1, 256) * big
    x[2] = torch.linspace(-1, 1, 256) * small
    x[3] = small * torch.finfo(t).eps * torch.arange(256)  # subnormals
    x[4, 5] = big
    x[4, 6] = small
    x[5, 100] = -small
    x[6] = 2.0 ** torch.linspace(-126, 127, 256)
    check_quantized(ms().quantize(x.cuda(), fmt), x, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_blocks_that_are_not_finite_read_back_as_nan(fmt):
    x = data(5, 128, torch.float32)
    x[0, 3], x[1, 40], x[2, 127] = float("nan"), float("inf"), -float("inf")
    t = ms().quantize(x, fmt)
    check_quantized(t, x, fmt)
    y = f64(ms().dequantize(t))
    b = O.BLOCK[fmt]
    for r, c in ((0, 3), (1, 40), (2, 127)):
        assert np.isnan(y[r, c // b * b:(c // b + 1) * b]).all()
    assert np.isnan(y).sum() == 3 * b


@pytest.mark.parametrize("g", [0.0, -1.0, float("nan"), float("inf")])
def test_a_tensor_scale_that_is_none_is_loud(g):
    t = ms().quantize(data(2, 64), "nvfp4", tensor_scale=torch.tensor([g], device="cuda"))
    assert torch.isnan(ms().dequantize(t, torch.float32)).all()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
def test_tensor_scale(dtype):
    for m, k, cut in ((1, 1, 0), (300, 777, 3), (1000, 6144, 0)):
        x = data(m, k, DTYPES[dtype], seed=k, cut=cut)
        got = ms().tensor_scale(x)
        assert got.dtype == torch.float32 and got.shape == (1,)
        # numpy divides as IEEE does; torch multiplies by the rounded reciprocal of a Python number
        assert np.float32(got.item()) == np.float32(x.abs().max().item()) / np.float32(2688)
    assert ms().tensor_scale(torch.zeros(4, 64, device="cuda")).item() == 1.0
    assert ms().tensor_scale(torch.zeros(0, 64, device="cuda")).item() == 1.0
    x[3, 5] = float("nan")
    assert torch.isnan(ms().tensor_scale(x)).all()


# ------------------------------------------------------------------ products
@pytest.mark.parametrize("a_fmt,w_fmt", PRODUCTS)
@pytest.mark.parametrize("m,n,k,dtype", [(1, 1, 1, "fp32"), (1, 128, 256, "fp32"), (2, 129, 300, "bf16"), (16, 500, 2048, "fp16"),
                                         (17, 64, 129, "fp32"), (33, 1537, 1030, "fp32"), (64, 8, 640, "bf16"),
                                         (65, 256, 128, "fp32"), (128, 1536, 384, "bf16"), (129, 257, 900, "fp32"),
                                         (300, 640, 1000, "fp16"), (1000, 520, 512, "bf16"), (513, 1100, 2047, "fp32")])
def test_product(a_fmt, w_fmt, m, n, k, dtype):
    q = ms().quantize
    ga = torch.tensor([0.037], device="cuda") if a_fmt == "nvfp4" else None
    x, w = data(m, k, seed=m), data(n, k, seed=n + 1, scale=0.05)
    a = q(x, a_fmt, tensor_scale=ga)
    wq = q(w, w_fmt, tensor_scale=ms().tensor_scale(w) if w_fmt == "nvfp4" else None)
    bias = data(1, n, torch.bfloat16, seed=9)[0].contiguous() if m % 2 else None
    y = ms().matmul(a, wq, bias, out_dtype=DTYPES[dtype])
    assert y.dtype == DTYPES[dtype]
    check_product(y, operand_values(a), operand_values(wq), bias, DTYPES[dtype])
    assert torch.equal(y, ms().matmul(a, wq, bias, out_dtype=DTYPES[dtype]))
    no_device_error()


@pytest.mark.parametrize("a_fmt,w_fmt", PRODUCTS)
@pytest.mark.parametrize("m", [3, 200, 700])
def test_nan_blocks_stay_in_their_rows(a_fmt, w_fmt, m):
    x, w = data(m, 520), data(300, 520, seed=2)
    clean = ms().matmul(ms().quantize(x, a_fmt), ms().quantize(w, w_fmt), out_dtype=torch.float32)
    x[1, 7], x[m - 1, 519], w[299, 100] = float("nan"), float("inf"), float("nan")
    y = ms().matmul(ms().quantize(x, a_fmt), ms().quantize(w, w_fmt), out_dtype=torch.float32)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[1], bad[m - 1], bad[:, 299] = True, True, True
    assert torch.equal(torch.isnan(y), bad)
    assert torch.equal(y[~bad], clean[~bad])


def test_product_writes_only_its_rows():
    """An output with a wider row stride: the columns past N stay as they were."""
    from krea2_svdquant_b200 import _lib, ops
    for m, n, k in ((5, 100, 256), (300, 520, 512)):
        a, w = ms().quantize(data(m, k), "mxfp4"), ms().quantize(data(n, k, seed=1), "mxfp4")
        out = torch.full((m + 1, n + 24), 7.0, device="cuda")
        _lib.call("svdq_mx_gemm", a.codes.data_ptr(), a.scales.data_ptr(), 1, None, w.codes.data_ptr(),
                  w.scales.data_ptr(), 1, None, None, out.data_ptr(), _lib.SVDQ_FP32, n + 24, m, n, k,
                  ops._raw_stream(out.device))
        assert (out[:, n:] == 7).all() and (out[m] == 7).all()
        check_product(out[:m, :n], operand_values(a), operand_values(w), None, torch.float32)


# ------------------------------------------------------------------ norm
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("m,h,cut", [(1, 1, 0), (1, 6144, 0), (130, 31, 1), (7, 1111, 0), (5, 2048, 8), (9, 2056, 0),
                                     (6, 4097, 3), (4, 8192, 0), (3, 16384, 0), (2, 20001, 0)])
@pytest.mark.parametrize("residual", [True, False])
def test_rms_norm(dtype, m, h, cut, residual):
    t = DTYPES[dtype]
    x, r = data(m, h, t, seed=1, cut=cut), data(m, h, t, seed=2)
    w = (data(1, h, torch.float32, seed=3)[0] * 0.1 + 1).to(t) if h % 2 else None
    q, total = ms().rms_norm(x, w, residual=r if residual else None, eps=1e-5)
    if residual:
        assert torch.equal(total, x + r)  # torch adds in fp32 and rounds once, as the kernel
    else:
        assert total is x
    y = O.rms_norm(f64(total), None if w is None else f64(w), 1e-5)
    # fp32: the mean's h additions, the root, two products: below (h + 8) 2^-24 relative; then one rounding to
    # e4m3 (half a step: 2^-4 relative, 2^-10 of the scale below its normal range), clipped at 448 scales
    byte = q.scales.cpu().numpy()[O.scale_index(m, O.k_pad(h) // 32)]
    s = np.repeat(O.E8M0[byte], 32, 1)[:, :h]
    got = operand_values(q)
    near = (h + 8) * 2.0 ** -24
    bound = np.maximum(np.abs(y) * 2.0 ** -4, s * 2.0 ** -10) + np.maximum(np.abs(y) - 448 * s, 0) + near * np.abs(y) * 2
    assert (np.abs(got - y) <= bound).all()
    ref_codes, ref_byte = O.quantize(y, "mxfp8")
    assert (byte != ref_byte).mean() <= 0.01  # amax next to a power of two
    assert (code_bytes(q) != ref_codes).mean() <= 0.01
    assert code_bytes(q)[:, h:].max(initial=0) == 0
    rest = np.ones(q.scales.numel(), bool)
    rest[O.scale_index(m, O.k_pad(h) // 32).ravel()] = False
    assert not q.scales.cpu().numpy()[rest].any()


def test_rms_norm_rows_that_are_zero_or_not_finite():
    x = data(4, 300)
    x[0] = 0
    x[1, 5] = float("nan")
    x[2, 299] = float("inf")
    q, _ = ms().rms_norm(x)
    y = ms().dequantize(q, torch.float32)
    assert (y[0] == 0).all() and torch.isnan(y[1]).all() and torch.isfinite(y[3]).all()
    assert torch.isnan(y[2, 288:]).all()  # inf / inf; the other columns are finite / inf
    assert (y[2, :288] == 0).all()


# ------------------------------------------------------------------ together, as they are used
@pytest.mark.parametrize("m", [1, 40, 333])
def test_norm_feeds_layers_that_share_it(m):
    """rms_norm -> three layers on its mxfp8 output, the sum feeding the next norm."""
    M = ms()
    x, r = data(m, 512, torch.bfloat16), data(m, 512, torch.bfloat16, seed=1)
    layers = [torch.nn.Linear(512, n, dtype=torch.bfloat16, device="cuda") for n in (512, 128, 256)]
    mx = [M.MicroscaledLinear.from_linear(l, act="mxfp8") for l in layers]
    h, total = M.rms_norm(x, residual=r)
    a = operand_values(h)
    ys = [l(h) for l in mx]
    for l, y in zip(mx, ys):
        check_product(y, a, operand_values(l.weight), l.bias, torch.bfloat16)
    h2, total2 = M.rms_norm(ys[0], residual=total)
    assert torch.equal(total2, ys[0] + total)
    check_product(mx[1](h2), operand_values(h2), operand_values(mx[1].weight), mx[1].bias, torch.bfloat16)
    no_device_error()


@pytest.mark.parametrize("act", ["nvfp4", "mxfp4", "mxfp8"])
def test_linear_quantises_on_the_way(act):
    M = ms()
    layer = torch.nn.Linear(700, 300, device="cuda")
    g = torch.tensor([0.02], device="cuda") if act == "nvfp4" else None
    lin = M.MicroscaledLinear.from_linear(layer, act=act, act_scale=g)
    x = data(60, 700).reshape(3, 20, 700)
    y = lin(x)
    assert y.shape == (3, 20, 300) and y.dtype == torch.float32
    a = M.quantize(x, act, tensor_scale=g)
    check_product(y.reshape(60, 300), operand_values(a), operand_values(lin.weight), lin.bias, torch.float32)
    assert torch.equal(M.linear(a, lin.weight, lin.bias, out_dtype=torch.float32), y)
    assert M.dequantize(a).shape == x.shape


@pytest.mark.parametrize("act", ["mxfp8", "nvfp4", "mxfp4"])
def test_stand_in_model(act):
    """The stand-in transformer on block-scaled linears: every layer's output against 64 bits on the
    operands that it received, and the layers behind a norm share one quantised input."""
    from krea2_svdquant_b200.transformer import Krea2StandInConfig, Krea2StandInTransformer
    M = ms()
    cfg = Krea2StandInConfig(num_layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, mlp=512, in_channels=32,
                             image_tokens=60, text_tokens=21)
    model = Krea2StandInTransformer.random_microscaled(cfg, act=act, seed=3)
    seen = {}
    for name, mod in model.named_modules():
        if isinstance(mod, M.MicroscaledLinear):
            mod.register_forward_hook(lambda m, a, y, name=name: seen.__setitem__(name, (m, a[0], y)))
    lat, txt = data(120, 32, torch.bfloat16).view(2, 60, 32), data(42, 256, torch.bfloat16).view(2, 21, 256)
    out = model(lat, txt)
    assert out.shape == (2, 60, 32) and torch.isfinite(out).all()
    assert len(seen) == 16
    for name, (mod, x, y) in seen.items():
        a = x if isinstance(x, M.MicroTensor) else M.quantize(x, act)
        check_product(y, operand_values(a), operand_values(mod.weight), mod.bias, torch.bfloat16)
    for i in range(2):
        p = f"transformer_blocks.{i}."
        shared = [seen[p + n][1] for n in ("attn.to_q", "attn.to_k", "attn.to_v", "attn.to_gate")]
        assert all(isinstance(s, M.MicroTensor) and s is shared[0] for s in shared)
        assert seen[p + "ff.gate"][1] is seen[p + "ff.up"][1]
    assert torch.equal(model(lat, txt), out)
    no_device_error()


def test_layers_move_and_keep_their_types():
    M = ms()
    lin = M.MicroscaledLinear.from_linear(torch.nn.Linear(130, 70, device="cuda"), act="nvfp4",
                                          act_scale=torch.tensor([0.1], device="cuda"))
    x = data(3, 130)
    y = lin(x)
    assert torch.equal(lin.half()(x), y) and lin.weight_scale.dtype == torch.float32 and lin.bias.dtype == torch.bfloat16
    assert torch.equal(lin.cpu().cuda()(x), y)
    other = M.MicroscaledLinear.from_linear(torch.nn.Linear(130, 70, device="cuda"), act="nvfp4",
                                            act_scale=torch.tensor([0.1], device="cuda"))
    other.load_state_dict(lin.state_dict())
    assert torch.equal(other(x), y)


def test_inputs_of_any_layout():
    """Transposed, expanded, sliced and higher-dimensional inputs."""
    M = ms()
    w = M.quantize(data(40, 96, seed=1), "mxfp4")
    base = data(96, 50)
    for x in (base.t(), base[:1].reshape(1, 1, 50).expand(3, 4, 50)[..., :1].expand(3, 4, 96),
              data(12, 200)[:, 7:103], data(24, 96).view(2, 3, 4, 96), data(10, 96)[::2]):
        dense = x.reshape(-1, 96).contiguous()
        want = M.linear(dense, w)
        assert torch.equal(M.linear(x, w).reshape(want.shape), want)
        for fmt in FORMATS:
            a, b = M.quantize(x, fmt), M.quantize(dense, fmt)
            assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)
        h, s = M.rms_norm(x, residual=x)
        h2, s2 = M.rms_norm(dense, residual=dense)
        assert torch.equal(h.codes.view(torch.uint8), h2.codes.view(torch.uint8)) and torch.equal(s.reshape(s2.shape), s2)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("offset", [1, 2, 3, 5, 8])
def test_rows_that_start_anywhere(dtype, offset):
    """Row starts at every alignment that the element type allows, at the end of an allocation too."""
    M, t = ms(), DTYPES[dtype]
    m, k = 9, 77
    flat = data(1, m * 83 + offset, t, seed=offset)[0]
    x = flat[offset:].view(m, 83)[:, 83 - k:]
    dense = x.contiguous()
    for fmt in FORMATS:
        a, b = M.quantize(x, fmt), M.quantize(dense, fmt)
        check_quantized(a, x, fmt)
        assert torch.equal(a.scales, b.scales)
    w = flat[offset:offset + k]
    h, s = M.rms_norm(x, w, residual=x)
    h2, s2 = M.rms_norm(dense, w.clone(), residual=dense)
    assert torch.equal(h.codes.view(torch.uint8), h2.codes.view(torch.uint8)) and torch.equal(s, s2)
    assert M.tensor_scale(x).item() == M.tensor_scale(dense).item()


def test_norm_in_place_through_the_c_abi():
    """sum may be x or the residual itself; columns past H of a wider sum stay as they were."""
    from krea2_svdquant_b200 import _lib, ops
    for h in (96, 101, 40000):
        x, r = data(5, h, torch.bfloat16), data(5, h, torch.bfloat16, seed=1)
        q, total = ms().rms_norm(x, residual=r)
        wide = torch.full((5, h + 11), 3.0, dtype=torch.bfloat16, device="cuda")
        wide[:, :h] = r
        codes, scales = torch.empty_like(q.codes), torch.empty_like(q.scales)
        _lib.call("svdq_rms_norm_mx", x.data_ptr(), h, wide.data_ptr(), h + 11, None, 0, 1e-6, 5, h, codes.data_ptr(),
                  scales.data_ptr(), wide.data_ptr(), h + 11, ops._raw_stream(x.device))
        assert torch.equal(wide[:, :h], total) and (wide[:, h:] == 3).all()
        assert torch.equal(codes.view(torch.uint8), q.codes.view(torch.uint8)) and torch.equal(scales, q.scales)


@pytest.mark.parametrize("act,w_fmt", PRODUCTS)
@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("m,n,k,cut", [(1, 128, 128, 0), (1, 300, 6144, 0), (3, 1537, 1030, 0), (2, 64, 77, 4), (4, 200, 640, 16),
                                       (4, 520, 2048, 0), (4, 129, 1, 2), (3, 2000, 999, 1), (5, 300, 700, 0)])
def test_few_tokens_quantised_by_the_product(act, w_fmt, dtype, m, n, k, cut):
    """Up to 4 tokens: one launch, the same bits as the quantisation and the product one after the other."""
    M = ms()
    x, w = data(m, k, DTYPES[dtype], seed=m, cut=cut), data(n, k, seed=n, scale=0.1)
    g = torch.tensor([0.0213], device="cuda") if act == "nvfp4" else None
    wq = M.quantize(w, w_fmt, tensor_scale=M.tensor_scale(w) if act == "nvfp4" else None)
    bias = data(1, n, torch.bfloat16, seed=3)[0].contiguous()
    a = M.quantize(x, act, tensor_scale=g)
    y = M.linear(x, wq, bias, act=act, act_scale=g)
    assert y.dtype == x.dtype and torch.equal(y, M.matmul(a, wq, bias, out_dtype=x.dtype))
    check_product(y, operand_values(a), operand_values(wq), bias, DTYPES[dtype])
    x[0, k // 2] = float("inf")
    y2 = M.linear(x, wq, bias, act=act, act_scale=g)
    assert torch.isnan(y2[0]).all() and torch.equal(y2[1:], y[1:])
    no_device_error()


@pytest.mark.parametrize("act,w_fmt", PRODUCTS)
@pytest.mark.parametrize("m", [4, 16, 64, 300])
def test_weight_written_just_before_the_call(act, w_fmt, m):
    """A weight that the launch before the linear writes (a quantisation, a copy) is the one it reads."""
    M = ms()
    x = data(m, 2048, torch.bfloat16)
    sources = [data(2000, 2048, torch.bfloat16, seed=i, scale=0.1) for i in range(3)]
    weights = [M.quantize(s, w_fmt) for s in sources]
    want = [M.matmul(M.quantize(x, act), w) for w in weights]
    torch.cuda.synchronize()
    w = M.MicroTensor(weights[0].codes.clone(), weights[0].scales.clone(), w_fmt, weights[0].shape)
    got, fresh = [], []
    for i in range(30):
        w.codes.copy_(weights[i % 3].codes)
        w.scales.copy_(weights[i % 3].scales)
        got.append(M.linear(x, w, act=act))
        fresh.append(M.linear(x, M.quantize(sources[i % 3], w_fmt), act=act))
    for i in range(30):
        assert torch.equal(got[i], want[i % 3]) and torch.equal(fresh[i], want[i % 3])
    no_device_error()


@pytest.mark.parametrize("m", [4, 16, 300])
def test_captured_with_the_weight_written_before(m):
    """A captured copy of the weight, or its quantisation, and the linear behind it, replayed with other weights."""
    M = ms()
    x, src = data(m, 1024, torch.bfloat16), data(1000, 1024, torch.bfloat16, seed=5, scale=0.1)
    w = M.quantize(src, "nvfp4")
    codes, graph = w.codes.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.codes.copy_(codes)
        copied = M.linear(x, w)
        fresh = M.linear(x, M.quantize(src, "nvfp4"))
    for i in range(10):
        codes.copy_(torch.roll(codes, 1, 0))
        src.copy_(torch.roll(src, 1, 1))
        graph.replay()
        assert torch.equal(copied, M.matmul(M.quantize(x, "nvfp4"), M.MicroTensor(codes, w.scales, "nvfp4", w.shape)))
        assert torch.equal(fresh, M.matmul(M.quantize(x, "nvfp4"), M.quantize(src, "nvfp4")))
    no_device_error()


def test_registered_ops():
    """The operators as torch custom ops: the same results, shapes under fake tensors, and a compiled call."""
    from krea2_svdquant_b200 import ops
    from torch._subclasses.fake_tensor import FakeTensorMode
    M, e, o = ms(), ops.eager, torch.ops.svdq_b200
    x, w = data(20, 300, torch.bfloat16), data(70, 300, seed=1)
    wq = M.quantize(w, "mxfp4")
    calls = {"mx_quantize": (x, "mxfp8", None), "mx_tensor_scale": (x,), "rms_norm_mx": (x, None, x, 1e-6),
             "mx_dequantize": (wq.codes, wq.scales, "mxfp4", 300, None, torch.float16),
             "mx_linear": (x, "mxfp8", None, wq.codes, wq.scales, "mxfp4", None, None, torch.bfloat16)}
    a = M.quantize(x, "mxfp4")
    calls["mx_gemm"] = (a.codes, a.scales, "mxfp4", None, wq.codes, wq.scales, "mxfp4", None, 300, None, torch.float32)
    for name, args in calls.items():
        got, want = getattr(o, name)(*args), getattr(e, name)(*args)
        got, want = (r if isinstance(r, (list, tuple)) else (r,) for r in (got, want))
        with FakeTensorMode() as mode:
            fake = getattr(o, name)(*[mode.from_tensor(v) if isinstance(v, torch.Tensor) else v for v in args])
        fake = fake if isinstance(fake, (list, tuple)) else (fake,)
        for g, r, f in zip(got, want, fake, strict=True):
            assert torch.equal(g.view(torch.uint8), r.view(torch.uint8))
            assert (f.shape, f.dtype) == (r.shape, r.dtype)
    run = lambda v: M.linear(M.rms_norm(v, residual=v)[0], wq) + M.linear(v, wq, act="mxfp8")
    assert torch.equal(torch.compile(run, fullgraph=True, backend="aot_eager")(x), run(x))


def test_empty_batches():
    M = ms()
    w = M.quantize(data(64, 128), "nvfp4")
    x = torch.empty(0, 128, device="cuda")
    for fmt in FORMATS:
        assert M.dequantize(M.quantize(x, fmt)).shape == (0, 128)
    assert M.linear(x, w).shape == (0, 64)
    q, s = M.rms_norm(x, residual=x)
    assert q.codes.shape == (0, 128) and s.shape == (0, 128)


def test_side_streams_and_captured_calls():
    """The same calls on two side streams at once and in two captured graphs, replayed in turn."""
    M = ms()
    w = M.MicroscaledLinear.from_linear(torch.nn.Linear(512, 384, dtype=torch.bfloat16, device="cuda"), act="nvfp4")
    xs = [data(m, 512, torch.bfloat16, seed=m) for m in (4, 300)]
    want = [w(x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for s, x in zip(streams, xs):
        with torch.cuda.stream(s):
            got.append([w(x) for _ in range(20)])
    torch.cuda.synchronize()
    for ys, y in zip(got, want):
        assert all(torch.equal(v, y) for v in ys)
    graphs, outs, ins = [], [], [x.clone() for x in xs]
    for x in ins:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            q, total = M.rms_norm(x, residual=x)
            outs.append((w(x), q.codes, total))
        graphs.append(g)
    for _ in range(3):
        for x in ins:
            x.mul_(0.5)
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for x, (y, codes, total) in zip(ins, outs):
        assert torch.equal(y, w(x)) and torch.equal(total, x + x)
        assert torch.equal(codes.view(torch.uint8), M.rms_norm(x, residual=x)[0].codes.view(torch.uint8))
    no_device_error()


def test_rows_past_two_to_the_31_elements():
    """A matrix of more than 2^31 elements: the last rows quantise and read back like rows of their own."""
    m, k = 140000, 16384
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB free")
    x = torch.zeros(m, k, dtype=torch.bfloat16, device="cuda")
    x[-3:] = data(3, k, torch.bfloat16)
    t = ms().quantize(x, "nvfp4")
    y = ms().dequantize(t)
    assert torch.equal(y[-3:], ms().dequantize(ms().quantize(x[-3:], "nvfp4")))
    assert not y[:-3].any()
    w = ms().quantize(data(64, k, seed=4), "nvfp4")
    p = ms().matmul(t, w)
    assert torch.equal(p[-3:], ms().matmul(ms().quantize(x[-256:], "nvfp4"), w)[-3:]) and not p[:-3].any()
