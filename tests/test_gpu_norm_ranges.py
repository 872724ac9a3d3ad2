"""The norm to mxfp8 on rows at the ends of the types' ranges, against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def rows(m, h, dtype, scale, seed=0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, h, generator=g, dtype=torch.float64).clamp(-3, 3) * scale).to(dtype).cuda()


def check(x, w, eps, residual=None):
    """Codes and scales of the norm of x against the definition in 64 bits.  y is within a few 2^-23 (relative) of
    it, one rounding to e4m3 is half a step: 2^-4 relative, 2^-10 of the scale below its normal range;
    magnitudes above 448 scales are clipped; a block's scale is that of a largest magnitude within 2^-20."""
    from krea2_svdquant_b200 import microscale as M
    q, total = M.rms_norm(x, w, residual=residual, eps=eps)
    m, h = x.shape
    y = O.rms_norm(f64(total), None if w is None else f64(w), eps)
    byte = q.scales.cpu().numpy()[O.scale_index(m, O.k_pad(h) // 32)]
    got = O.values(O.unpack(q.codes.view(torch.uint8).cpu().numpy(), "mxfp8"), byte, "mxfp8")[:, :h]
    s = np.repeat(O.E8M0[byte], 32, 1)[:, :h]
    assert np.isfinite(got).all()
    assert (np.abs(got - y) <= np.maximum(np.abs(y) * 2.0 ** -4, s * 2.0 ** -10)
            + np.maximum(np.abs(y) - 448 * s, 0) + 2.0 ** -20 * np.abs(y)).all()
    for near in (1 - 2.0 ** -20, 1 + 2.0 ** -20):  # the scale of a block is that of y or of a y next to it
        ref = O.quantize(y * near, "mxfp8")[1]
        byte = np.where(byte == ref, 0, byte)
    assert not byte.any()


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("h", [17, 256, 1111, 6144, 20001])
@pytest.mark.parametrize("scale,eps", [(1e19, 1e-6), (1e25, 1e-6), (1e38, 1e-6), (1e25, 0.0), (1e-12, 0.0), (1e-23, 0.0),
                                       (1e-25, 0.0), (1e-37, 0.0), (1.0, 1e30), (1e18, 1e38)])
def test_rows_far_from_one(dtype, h, scale, eps):
    x = rows(5, h, DTYPES[dtype], scale, seed=h)
    x[2, 1:] = 0  # one element that is not zero
    check(x, None, eps)
    check(x, rows(1, h, DTYPES[dtype], 1.0, seed=1)[0], eps)


@pytest.mark.parametrize("h", [40, 2048, 20001])
def test_rows_of_subnormal_numbers(h):
    x = rows(4, h, torch.float32, 1e-41)
    check(x, None, 0.0)
    x = rows(4, h, torch.bfloat16, 3e-39)
    check(x, None, 0.0)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("h", [48, 1111, 6144, 20001])
@pytest.mark.parametrize("scale,weight,eps", [(1e30, 1e12, 1e-6), (1e18, 1e25, 1e-6), (1e-22, 1e-25, 0.0), (1e-25, 1e30, 1e-6),
                                              (1e-17, 1e-25, 1e-38), (1.0, 1e-30, 1e-6), (1e-20, 1e-12, 1e-6)])
def test_weights_far_from_one(dtype, h, scale, weight, eps):
    """x * weight is past the range of fp32 where the norm is not."""
    t = DTYPES[dtype]
    check(rows(4, h, t, scale, seed=2), rows(1, h, t, weight, seed=3)[0], eps)


def test_ranges_meet_in_one_matrix():
    """Ordinary rows between rows of other ranges, with a residual; columns of weights of every size."""
    h = 1536
    x = torch.cat([rows(3, h, torch.float32, s, seed=i) for i, s in enumerate((1.0, 1e30, 1e-30, 0.0, 1e-3, 1e10))])
    check(x, None, 1e-6)
    check(x, None, 1e-6, residual=x.flip(0).contiguous())
    w = 10.0 ** torch.linspace(-30, 30, h, dtype=torch.float64).to(torch.float32).cuda()
    check(x, w, 1e-6)
    y = rows(2, h, torch.float32, 1.0)
    y[:, 64:128] = 0  # whole blocks of zeros
    check(y, None, 1e-6)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("h", [1, 40, 300, 1111, 20001])
def test_padding_of_rows_without_a_norm(dtype, h):
    """Zeros without eps (0 / 0), an infinity, a NaN: the row's own blocks are NaN where the norm is, those that fill it
    up to 128 columns hold zeros."""
    from krea2_svdquant_b200 import microscale as M
    x = torch.ones(5, h, device="cuda", dtype=dtype)
    x[0] = 0
    x[1, h // 2] = float("nan")
    x[2, h // 2] = float("inf")
    for w in (None, torch.ones(h, device="cuda", dtype=dtype)):
        q, _ = M.rms_norm(x, w, eps=0.0)
        byte = torch.from_numpy(q.scales.cpu().numpy()[O.scale_index(5, O.k_pad(h) // 32)])
        own = -(-h // 32)
        assert (byte[:2, :own] == 255).all() and (byte[:, own:] == 0).all()
        assert byte[2, h // 64] == 255 and (byte[2, :own] == 255).sum() == 1
        assert (byte[3:, :own] == 119).all()  # 2^-8: a norm of ones
        assert not q.codes.view(torch.uint8)[:, h:].any()
