"""nvfp4 from fp32: numbers next to every kind of border, with many tensor scales, against exact arithmetic."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu

E2M1_MID = (O.E2M1[1:8] + O.E2M1[:7]) / 2
E4M3_MID = (O.E4M3[1:127] + O.E4M3[:126]) / 2


def check(x: np.ndarray, g: np.float32):
    """Scales and codes of x [rows, K] bit for bit.  The oracle's quotients in 64 bits are exact enough: x / (scale g)
    differs from a border, if at all, by 2^-31 of it or more (24 + 28 + 3 bits), amax / (6 g) by 2^-33."""
    from krea2_svdquant_b200 import microscale as M
    x = torch.from_numpy(np.ascontiguousarray(x, np.float32)).cuda()
    t = M.quantize(x, "nvfp4", tensor_scale=torch.tensor([g], device="cuda"))
    codes, byte = O.quantize(x.double().cpu().numpy(), "nvfp4", float(g))
    np.testing.assert_array_equal(t.scales.cpu().numpy()[O.scale_index(len(x), byte.shape[1])], byte)
    np.testing.assert_array_equal(O.unpack(t.codes.cpu().numpy(), "nvfp4"), codes)


def beside(v: np.ndarray) -> np.ndarray:
    """The fp32 number nearest to each v and its two neighbours, [..., 3]."""
    f = v.astype(np.float32)
    return np.stack((np.nextafter(f, np.float32(0)), f, np.nextafter(f, np.float32(np.inf))), -1)


def test_known_numbers():
    """Two that a quotient rounded to fp32 puts on the wrong side: x / (scale g) = 1.7499999985 is code 3 (1.5), and
    amax / (6 g) = 1.6875000084 is scale 1.75."""
    bits = lambda u: np.array([u], np.uint32).view(np.float32)[0]
    g, unit = bits(0x3AAC1259), O.E4M3[15]
    x = np.zeros((1, 16), np.float32)
    x[0, 0], x[0, 1], x[0, 2] = np.float32(6 * unit * g), bits(0x388D270D), -bits(0x388D270D)
    check(x, g)
    x[0] = 0
    x[0, 3] = bits(0x418FE94D)
    check(x, bits(0x3FE36A5A))


@pytest.mark.parametrize("seed", range(8))
def test_codes_next_to_their_borders(seed):
    """The numbers next to every border of every scale, for 24 tensor scales of 24 bits each."""
    rng = np.random.default_rng(seed)
    sf = O.E4M3[9:127]
    for _ in range(24):
        g = np.float32(rng.uniform(0.5, 1) * 2.0 ** rng.integers(-30, 30))
        unit = sf * np.float64(g)
        near = beside(unit[:, None] * E2M1_MID).reshape(len(sf), -1)  # 21 a scale
        top = (unit * 6).astype(np.float32)[:, None]                  # fixes the block's scale
        check(np.concatenate([top, near[:, :15], -top, near[:, 6:]], 1), g)


@pytest.mark.parametrize("seed", range(8))
def test_scales_next_to_their_borders(seed):
    """Largest elements next to every border between two scales, for 200 tensor scales."""
    rng = np.random.default_rng(100 + seed)
    for _ in range(200):
        g = np.float32(rng.uniform(0.5, 1) * 2.0 ** rng.integers(-30, 30))
        amax = beside(6 * np.float64(g) * E4M3_MID).reshape(-1)
        x = np.zeros((amax.size, 16), np.float32)
        x[np.arange(amax.size), rng.integers(0, 16, amax.size)] = amax * rng.choice([-1, 1], amax.size)
        check(x, g)


@pytest.mark.parametrize("lo,hi", [(-126, -90), (-90, -60), (60, 90), (90, 110)])
def test_tensor_scales_at_the_ends(lo, hi):
    """Tensor scales where the quotients change from fp32 to 64 bits."""
    rng = np.random.default_rng(7)
    sf = O.E4M3[40:100]
    for _ in range(20):
        g = np.float32(rng.uniform(0.5, 1) * 2.0 ** rng.integers(lo, hi))
        unit = sf * np.float64(g)
        near = beside(unit[:, None] * E2M1_MID).reshape(len(sf), -1)
        check(np.concatenate([(unit * 6).astype(np.float32)[:, None], near[:, :15]], 1), g)
        amax = beside(6 * np.float64(g) * E4M3_MID[40:100]).reshape(-1)
        x = np.zeros((amax.size, 16), np.float32)
        x[:, 5] = amax
        check(x, g)
