"""The norm's codes and scales are those of its exact value: bit for bit against 64 bits."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().double().cpu().numpy()


def check(x, w, eps, residual=None):
    """The oracle's y is within some 2^-50 of the exact one, so a code can differ only where a border is as near,
    which the inputs of these tests do not come to (one in 10^13 would)."""
    from krea2_svdquant_b200 import microscale as M
    q, total = M.rms_norm(x, w, residual=residual, eps=eps)
    m, h = x.shape
    codes, byte = O.quantize(O.rms_norm(f64(total), None if w is None else f64(w), eps), "mxfp8")
    np.testing.assert_array_equal(q.scales.cpu().numpy()[O.scale_index(m, O.k_pad(h) // 32)], byte)
    np.testing.assert_array_equal(O.unpack(q.codes.view(torch.uint8).cpu().numpy(), "mxfp8"), codes)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("m,h,cut", [(600, 6144, 0), (150, 8192, 8), (300, 4097, 3), (40, 20001, 0), (2000, 333, 0), (5, 31, 1)])
@pytest.mark.parametrize("residual", [True, False])
def test_every_code_is_that_of_the_exact_norm(dtype, m, h, cut, residual):
    """Values with outlier columns, some of whose norms lie within fp32's rounding of a border."""
    g = torch.Generator(device="cuda").manual_seed(h + cut)
    t = DTYPES[dtype]

    def values():
        v = torch.randn(m, h + cut, generator=g, device="cuda")
        v[:, ::53] *= 20
        return v.to(t)[:, :h]

    x, r = values(), values() if residual else None
    w = (1 + 0.1 * torch.randn(h, generator=g, device="cuda")).to(t)
    check(x, w, 1e-6, r)
    check(x, None, 1e-5, r)


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("c", [1.0, 0.75, 3.0, 1.1, 0.013, 240.0])
def test_norms_that_lie_on_borders(dtype, c):
    """Rows of equal magnitudes without eps: the norm is exactly the weight, here every border between codes
    (ties to even), its neighbours, and powers of two as a block's largest value."""
    t = DTYPES[dtype]
    table = O.E4M3[1:127]
    w = np.concatenate([(table[1:] + table[:-1]) / 2, table]) / 256
    w = torch.from_numpy(np.resize(w, 512)).to(t)
    near = torch.cat([w, torch.nextafter(w, torch.zeros_like(w)), torch.nextafter(w, w * 2)])
    w = near[torch.randperm(near.numel(), generator=torch.Generator().manual_seed(1))].cuda()
    x = torch.full((4, w.numel()), c, device="cuda").to(t)
    x[1] *= -1
    x[2, ::3] *= -1
    check(x, w, 0.0)
    check(x, torch.ones_like(w), 0.0)
    check(x, w, 1e-6)


def test_a_long_row():
    """2^20 columns: a sum of their squares in 32 bits would be off by more than a step of the last bit."""
    h = 1 << 20
    x = torch.full((2, h), 1.1, device="cuda")
    x[1, ::3] = -1.7
    w = torch.full((h,), 1.0 + 2.0 ** -3 + 2.0 ** -4, device="cuda")  # a border between two codes
    for eps in (0.0, 4e-7, 1e-6):
        check(x, w, eps)


def test_zeros_keep_their_codes():
    """Rows and columns of zeros of both signs beside ordinary ones."""
    x = torch.randn(64, 777, generator=torch.Generator().manual_seed(4)).cuda()
    x[:, ::2] = 0.0
    x[:, 1::6] = -0.0
    x[5], x[6] = 0.0, -0.0
    for t in DTYPES.values():
        check(x.to(t), None, 1e-6)
        check(x.to(t), torch.full((777,), -1.3, device="cuda").to(t), 1e-6)
