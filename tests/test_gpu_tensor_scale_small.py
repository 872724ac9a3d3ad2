"""The nvfp4 tensor scale of matrices near the small end of fp32."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu


AMAX = [2.0 ** -149, 1.5e-42, 1.8e-42, 4.0e-42, 1e-40, 1e-38, 3.1e-35, 3.2e-35, 1e-34]


@pytest.mark.parametrize("dtype,amax", [(t, a) for t in (torch.float32, torch.bfloat16) for a in AMAX
                                        if a >= torch.finfo(t).smallest_normal * torch.finfo(t).eps])
def test_small_matrices_keep_their_values(dtype, amax):
    """A positive scale, no smaller than amax / 2688, so that nothing saturates or turns to NaN; codes by the definition."""
    from krea2_svdquant_b200 import microscale as M
    x = (torch.linspace(-1, 1, 4 * 256, dtype=torch.float64) * amax).to(dtype).view(4, 256)
    x[0, 0] = amax
    top = x.abs().max().item()
    g = M.tensor_scale(x.cuda())
    v = np.float32(g.item())
    exact = np.float64(top) / 2688
    if exact >= 2.0 ** -126:
        assert v == np.float32(np.float32(top) / np.float32(2688))
    else:  # rounded up to a multiple of the smallest number
        assert float(v) == np.ceil(exact * 2.0 ** 149) * 2.0 ** -149 and v > 0
    t = M.quantize(x.cuda(), "nvfp4", tensor_scale=g)
    codes, byte = O.quantize(x.double().numpy(), "nvfp4", float(v))
    np.testing.assert_array_equal(t.scales.cpu().numpy()[O.scale_index(4, byte.shape[1])], byte)
    np.testing.assert_array_equal(O.unpack(t.codes.cpu().numpy(), "nvfp4"), codes)
    y = M.dequantize(t, torch.float32).double().cpu().numpy()
    # code * fl(scale * g): half a step of the code, and half of the smallest number six times for the unit
    unit = np.repeat(O.E4M3[byte], 16, 1) * float(v)
    assert (np.abs(y - x.double().numpy()) <= unit * 1.0 + 6.5 * 2.0 ** -149 + np.maximum(np.abs(x.double().numpy()) - 6 * unit, 0)).all()
