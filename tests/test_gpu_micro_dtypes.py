"""Block-scaled layers keep the type of the values that were quantised for them."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("act", ["nvfp4", "mxfp4", "mxfp8"])
def test_a_quantised_input_gives_what_its_values_give(dtype, act):
    from krea2_svdquant_b200 import microscale as M
    t = DTYPES[dtype]
    lin = M.MicroscaledLinear.from_linear(torch.nn.Linear(256, 130, device="cuda"), act=act)
    x = torch.randn(33, 256, device="cuda").to(t)
    y, shared = lin(x), lin(M.quantize(x, act))
    assert y.dtype == t and shared.dtype == t and torch.equal(y, shared)
    h, total = M.rms_norm(x, residual=x)
    assert h.dtype == t and total.dtype == t
    if act == "mxfp8":
        assert lin(h).dtype == t
    a = M.quantize(x, act)
    assert M.linear(a, lin.weight, out_dtype=torch.float32).dtype == torch.float32
    unknown = M.MicroTensor(a.codes, a.scales, a.fmt, a.shape)
    assert M.linear(unknown, lin.weight).dtype == torch.bfloat16


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("act", ["nvfp4", "mxfp4", "mxfp8"])
def test_stand_in_model_of_every_type(dtype, act):
    """Every layer's output, the shared ones' too, in the model's type, and the product of what went in."""
    from krea2_svdquant_b200 import microscale as M
    from krea2_svdquant_b200.transformer import Krea2StandInConfig, Krea2StandInTransformer
    t = DTYPES[dtype]
    cfg = Krea2StandInConfig(num_layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, mlp=512, in_channels=32,
                             image_tokens=60, text_tokens=21)
    model = Krea2StandInTransformer.random_microscaled(cfg, act=act, seed=3, dtype=t)
    seen = []
    for mod in model.modules():
        if isinstance(mod, M.MicroscaledLinear):
            mod.register_forward_hook(lambda m, a, y: seen.append((m, a[0], y)))
    g = torch.Generator(device="cuda").manual_seed(1)
    lat = torch.randn(2, 60, 32, generator=g, device="cuda").to(t)
    txt = torch.randn(2, 21, 256, generator=g, device="cuda").to(t)
    out = model(lat, txt)
    assert out.dtype == t and torch.isfinite(out).all() and len(seen) == 16
    assert sum(isinstance(x, M.MicroTensor) for _, x, _ in seen) == 12
    for mod, x, y in seen:
        a = x if isinstance(x, M.MicroTensor) else M.quantize(x, act)
        assert y.dtype == t
        assert torch.equal(y.reshape(-1, y.shape[-1]), M.matmul(a, mod.weight, mod.bias, out_dtype=t).reshape(-1, y.shape[-1]))
