"""Block-scaled products with several tiles to each pair of CTAs: the accumulators in turn, their shared columns, the
ring across tiles, and row blocks in more than one group."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu

PRODUCTS = (("nvfp4", "nvfp4"), ("mxfp4", "mxfp4"), ("mxfp8", "mxfp4"))
TABLES = {"4": O.E2M1, "8": O.E4M3}


def operand(m, k, fmt, seed):
    """Random codes and scales, and the values they stand for in 64 bits on the GPU (without a quantisation, so that
    every element counts).  Scales of 2^-2 to 2^1, so that no product outgrows the others."""
    from krea2_svdquant_b200 import microscale as M, ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    kp, block = O.k_pad(k), O.BLOCK[fmt]
    n = 256 if fmt == "mxfp8" else 16
    code = torch.randint(0, n, (m, kp), generator=g, device="cuda")
    if fmt == "mxfp8":
        code = torch.where((code & 127) > 0x60, code ^ 0x60, code)  # no NaN, magnitudes up to 32
    code[:, k:] = 0
    e = torch.randint(-2, 2, (m, kp // block), generator=g, device="cuda")
    byte = ((e + 7) << 3 | torch.randint(0, 8, e.shape, generator=g, device="cuda")) if fmt == "nvfp4" else e + 127
    scales = torch.zeros(ops.mx_scales_numel(m, k, fmt), dtype=torch.uint8, device="cuda")
    r, c = torch.arange(m, device="cuda")[:, None], torch.arange(kp // block, device="cuda")[None, :]
    at = ((r // 128) * (kp // block // 4) + c // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + c % 4
    scales[at] = byte.to(torch.uint8)
    table = torch.from_numpy(TABLES["8" if fmt == "mxfp8" else "4"]).cuda()
    unit = torch.from_numpy(O.E4M3 if fmt == "nvfp4" else O.E8M0).cuda()[byte]
    values = (table[code].view(m, -1, block) * unit[..., None]).view(m, -1)[:, :k]
    if fmt == "mxfp8":
        codes = code.to(torch.uint8).view(torch.float8_e4m3fn)
    else:
        codes = (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8)
    return M.MicroTensor(codes.contiguous(), scales, fmt, (m, k)), values


def check(m, n, k, a_fmt, w_fmt, dtype, bias, wide=0):
    """Every element against 64 bits.  The tensor core adds in fp32 and may truncate: K additions of 2^-23 of the sum of
    magnitudes at most; alpha, bias and the output round by half a step each."""
    from krea2_svdquant_b200 import _lib, microscale as M, ops
    a, av = operand(m, k, a_fmt, 1)
    w, wv = operand(n, k, w_fmt, 2)
    b = (torch.randn(n, device="cuda") * 10).to(torch.bfloat16) if bias else None
    if wide:
        out = torch.full((m, n + wide), 3.0, dtype=dtype, device="cuda")
        _lib.call("svdq_mx_gemm", a.codes.data_ptr(), a.scales.data_ptr(), ops.MX_FORMATS[a_fmt], None, w.codes.data_ptr(),
                  w.scales.data_ptr(), ops.MX_FORMATS[w_fmt], None, None if b is None else b.data_ptr(), out.data_ptr(),
                  ops._DT[dtype], n + wide, m, n, k, ops._raw_stream(out.device))
        assert (out[:, n:] == 3).all()
        y = out[:, :n]
    else:
        y = M.matmul(a, w, b, out_dtype=dtype)
        assert torch.equal(y, M.matmul(a, w, b, out_dtype=dtype))
    ref, mag = av @ wv.t(), av.abs() @ wv.abs().t()
    if b is not None:
        ref, mag = ref + b.double(), mag + b.double().abs()
    u = torch.finfo(dtype).eps / 2
    near = (k + 3) * 2.0 ** -23 * mag
    bad = (y.double() - ref).abs() > near + u * (ref.abs() + near)
    assert not bad.any(), (int(bad.sum()), bad.nonzero()[:5].tolist())
    # errors do not line up: far closer than the bound on the whole
    assert (y.double() - ref).norm() <= (1e-5 + u) * ref.norm()
    assert _lib.device_error() == 0


@pytest.mark.parametrize("a_fmt,w_fmt", PRODUCTS)
@pytest.mark.parametrize("m,n,k,dtype,bias", [(2100, 6500, 200, "fp32", False), (2100, 6500, 1500, "bf16", True),
                                              (2048, 6400, 200, "bf16", False), (2304, 6656, 900, "fp16", True),
                                              (4352, 6144, 130, "fp32", True), (2561, 5001, 2048, "fp16", False)])
def test_three_and_more_tiles_a_pair(a_fmt, w_fmt, m, n, k, dtype, bias):
    """9 x 26 tiles and more on 74 pairs; one stage a tile and several; rows stored whole (N a multiple of 32
    bytes) and through shared memory."""
    check(m, n, k, a_fmt, w_fmt, {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}[dtype], bias)


@pytest.mark.parametrize("a_fmt,w_fmt", PRODUCTS)
@pytest.mark.parametrize("wide", [5, 16])
def test_outputs_with_a_row_stride(a_fmt, w_fmt, wide):
    check(2100, 6400, 700, a_fmt, w_fmt, torch.bfloat16, True, wide)


@pytest.mark.parametrize("a_fmt,w_fmt,m,k", [("nvfp4", "nvfp4", 9000, 8192), ("mxfp4", "mxfp4", 9000, 8192),
                                             ("mxfp8", "mxfp4", 5000, 8192)])
def test_row_blocks_in_groups(a_fmt, w_fmt, m, k):
    """Activations of more than 28 MB: two groups of row blocks, of 18 each (nvfp4, mxfp4) or 10, the last with rows
    missing."""
    check(m, 1300, k, a_fmt, w_fmt, torch.float32, False)


def test_groups_of_different_sizes():
    """71 row blocks in groups of 24, 24 and 23."""
    check(18100, 700, 6144, "nvfp4", "nvfp4", torch.bfloat16, True)


@pytest.mark.parametrize("a_fmt,w_fmt", PRODUCTS)
def test_many_tiles_one_after_the_other(a_fmt, w_fmt):
    """64 x 30 tiles of a single stage each: hand-offs as close together as they come."""
    check(16384, 7680, 64, a_fmt, w_fmt, torch.bfloat16, False)
