"""A calibrated stand-in model quantises each norm's output once, before and after its tensors move."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_calibrated_model_shares_after_moves():
    from krea2_svdquant_b200 import microscale as M
    from krea2_svdquant_b200.offload import enable_block_offload
    from krea2_svdquant_b200.transformer import Krea2StandInConfig, Krea2StandInTransformer
    cfg = Krea2StandInConfig(num_layers=2, hidden=256, heads=4, kv_heads=2, head_dim=64, mlp=512, in_channels=32,
                             image_tokens=60, text_tokens=21)
    model = Krea2StandInTransformer.random_microscaled(cfg, act="nvfp4", seed=3)
    for b in model.transformer_blocks:
        one, two = torch.tensor([0.002], device="cuda"), torch.tensor([0.003], device="cuda")
        for lin in (b.attn.to_q, b.attn.to_k, b.attn.to_v, b.attn.to_gate):
            lin.act_scale = one
        b.ff.gate.act_scale = b.ff.up.act_scale = two
    seen = []
    for mod in model.modules():
        if isinstance(mod, M.MicroscaledLinear):
            mod.register_forward_hook(lambda m, a, y: seen.append(a[0]))
    g = torch.Generator(device="cuda").manual_seed(1)
    lat = torch.randn(2, 60, 32, generator=g, device="cuda", dtype=torch.bfloat16)
    txt = torch.randn(2, 21, 256, generator=g, device="cuda", dtype=torch.bfloat16)

    def run():
        seen.clear()
        y = model(lat, txt)
        inputs = {id(x) for x in seen if isinstance(x, M.MicroTensor)}
        assert len(seen) == 16 and len(inputs) == 4 and sum(isinstance(x, M.MicroTensor) for x in seen) == 12
        return y

    want = run()
    model.cpu().cuda()
    assert torch.equal(run(), want)
    off = enable_block_offload(model, "cuda", num_blocks_on_gpu=1)
    assert torch.equal(run(), want) and torch.equal(run(), want)
    off.remove()
