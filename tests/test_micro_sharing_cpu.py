"""Layers that share an activation scale keep sharing it through moves, loads and the offloader."""
from __future__ import annotations

import torch

from krea2_svdquant_b200 import microscale as M, ops
from krea2_svdquant_b200.offload import _BlockArena
from krea2_svdquant_b200.transformer import Krea2StandInBlock, Krea2StandInConfig, _shared_format

CFG = Krea2StandInConfig(num_layers=1, hidden=128, heads=2, kv_heads=1, head_dim=64, mlp=256, in_channels=8, image_tokens=4,
                         text_tokens=2)


def block(scales):
    def make(name):
        n, k = CFG.linear_shapes()[name]
        w = M.MicroTensor(torch.zeros(n, ops.mx_k_pad(k) // 2, dtype=torch.uint8),
                          torch.zeros(ops.mx_scales_numel(n, k, "nvfp4"), dtype=torch.uint8), "nvfp4", (n, k), torch.ones(1))
        return M.MicroscaledLinear(w, act="nvfp4", act_scale=scales(name))
    return Krea2StandInBlock(CFG, make)


def shared(b):
    return [_shared_format(v) is not None for v in ((b.attn.to_q, b.attn.to_k, b.attn.to_v, b.attn.to_gate), (b.ff.gate, b.ff.up))]


def calibrated():
    one, two = torch.tensor([0.5]), torch.tensor([0.25])
    return block(lambda name: one if name.startswith("attn.to_") and "out" not in name else two)


def test_a_move_keeps_shared_scales_shared():
    b = calibrated()
    assert shared(b) == [True, True]
    state = {k: v.clone() for k, v in b.state_dict().items()}
    b.to("meta")
    assert shared(b) == [True, True] and b.attn.to_q.act_scale.device.type == "meta"
    b.to_empty(device="cpu")
    assert shared(b) == [True, True]
    b.load_state_dict(state)
    assert shared(b) == [True, True]
    assert b.attn.to_q.act_scale.item() == 0.5 and b.ff.up.act_scale.item() == b.ff.down.act_scale.item() == 0.25


def test_scales_of_their_own_stay_apart():
    b = block(lambda name: torch.tensor([0.5]))
    assert shared(b) == [False, False]
    b.to("meta")
    b.to_empty(device="cpu")
    assert shared(b) == [False, False]
    assert len({id(m.act_scale) for m in b.modules() if isinstance(m, M.MicroscaledLinear)}) == 8


def test_a_packed_block_keeps_shared_buffers_shared():
    b = calibrated()
    want = {k: v.clone() for k, v in b.state_dict().items()}
    arena = _BlockArena(b, pin=False)
    assert shared(b) == [True, True]
    base = torch.zeros_like(arena.host)
    base.copy_(arena.host)
    arena.attach_device(base)
    assert shared(b) == [True, True]
    assert b.attn.to_v.act_scale.untyped_storage().data_ptr() == base.untyped_storage().data_ptr()
    for k, v in b.state_dict().items():
        assert torch.equal(v, want[k])
    arena.attach_cpu()
    assert shared(b) == [True, True]
    arena.to_device_plain(torch.device("cpu"), False)
    assert shared(b) == [True, True]
