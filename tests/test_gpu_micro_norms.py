"""The stand-in block's shared quantised norm is that of the norm module: its hooks, its epsilon, its type."""
from __future__ import annotations

import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu


def model(act):
    from krea2_svdquant_b200.transformer import Krea2StandInConfig, Krea2StandInTransformer
    cfg = Krea2StandInConfig(num_layers=1, hidden=256, heads=4, kv_heads=2, head_dim=64, mlp=512, in_channels=32,
                             image_tokens=60, text_tokens=21)
    return Krea2StandInTransformer.random_microscaled(cfg, act=act, seed=3)


def data():
    g = torch.Generator(device="cuda").manual_seed(1)
    return (torch.randn(2, 60, 32, generator=g, device="cuda", dtype=torch.bfloat16),
            torch.randn(2, 21, 256, generator=g, device="cuda", dtype=torch.bfloat16))


@pytest.mark.parametrize("act", ["nvfp4", "mxfp4", "mxfp8"])
def test_hooks_of_a_norm_run(act):
    m, (lat, txt) = model(act), data()
    norms = [m.transformer_blocks[0].norm1, m.transformer_blocks[0].norm2]
    want, calls = m(lat, txt), []
    hooks = [n.register_forward_hook(lambda mod, a, y: calls.append(mod)) for n in norms]
    hooks += [n.register_forward_pre_hook(lambda mod, a: calls.append(mod)) for n in norms]
    m(lat, txt)
    assert calls == [norms[0]] * 2 + [norms[1]] * 2
    for h in hooks:
        h.remove()
    hook = norms[0].register_forward_hook(lambda mod, a, y: y * 0)  # a hook's output is what the layers read
    changed = m(lat, txt)
    hook.remove()
    assert not torch.equal(changed, want) and torch.equal(m(lat, txt), want)
    hook = nn.modules.module.register_module_forward_hook(lambda mod, a, y: calls.append(mod) if mod in norms else None)
    calls.clear()
    m(lat, txt)
    hook.remove()
    assert calls == norms


@pytest.mark.parametrize("act", ["nvfp4", "mxfp4", "mxfp8"])
def test_other_norm_modules(act):
    """A norm without an epsilon of its own or without a weight, one in another type, one of another class."""
    from krea2_svdquant_b200 import microscale as M
    from krea2_svdquant_b200.transformer import _quantized_norm

    class Half(nn.RMSNorm):
        def forward(self, x):
            return super().forward(x) * 0.5

    x = torch.randn(40, 256, device="cuda", dtype=torch.bfloat16) * 1e-2
    for norm in (nn.RMSNorm(256, device="cuda", dtype=torch.bfloat16), nn.RMSNorm(256, eps=1e-5, elementwise_affine=False),
                 nn.RMSNorm(256, eps=1e-5, device="cuda"), Half(256, eps=1e-5, device="cuda", dtype=torch.bfloat16)):
        h, total = _quantized_norm(norm, x, act, None, residual=x)
        want = norm((x + x)).float()
        assert torch.equal(total, x + x) and h.fmt == act
        got = M.dequantize(h, torch.float32)
        # of a block's largest magnitude: a quarter with 4 bits (half the step from 4 to 6, or 8 clipped to 6), an eighth
        # with 8 bits (512 clipped to 448), and 2^-8 for the module's own rounding to bf16
        top = want.abs().view(40, -1, M.ops.MX_BLOCK[act]).amax(-1, keepdim=True)
        err = (got - want).abs().view(top.shape[0], top.shape[1], -1)
        assert (err <= top * (0.26 if act != "mxfp8" else 0.13)).all()
