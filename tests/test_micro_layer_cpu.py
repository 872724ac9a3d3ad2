"""MicroscaledLinear's buffers under the moves and casts of a module, without a GPU."""
from __future__ import annotations

import pytest
import torch

from krea2_svdquant_b200 import microscale as M


def layer(act_scale=None, bias=True):
    w = M.MicroTensor(torch.arange(4 * 64, dtype=torch.uint8).view(4, 64), torch.arange(1024).to(torch.uint8), "nvfp4", (4, 100),
                      torch.tensor([0.3]))
    return M.MicroscaledLinear(w, torch.tensor([0.1, -2.0, 3.3, 1e30]) if bias else None, act="nvfp4", act_scale=act_scale)


@pytest.mark.parametrize("act_scale", [None, torch.tensor([0.7]), torch.tensor(0.7)])
@pytest.mark.parametrize("bias", [True, False])
def test_to_empty_of_a_layer_on_meta(act_scale, bias):
    """A layer made without memory, given some, and loaded."""
    lin = layer(act_scale, bias)
    empty = layer(act_scale, bias).to("meta")
    assert all(b.device.type == "meta" for b in empty.buffers())
    empty = empty.to_empty(device="cpu")
    assert all(b.device.type == "cpu" for b in empty.buffers())
    empty.load_state_dict(lin.state_dict())
    for (n, a), (m, b) in zip(lin.named_buffers(), empty.named_buffers(), strict=True):
        assert n == m and a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


@pytest.mark.parametrize("cast", [lambda m: m.half(), lambda m: m.double(), lambda m: m.to(torch.bfloat16),
                                  lambda m: m.to("cpu", torch.float16)])
def test_casts_leave_the_buffers_as_they_are(cast):
    lin, ref = layer(torch.tensor([0.7])), layer(torch.tensor([0.7]))
    cast(lin)
    for a, b in zip(lin.buffers(), ref.buffers(), strict=True):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_a_move_that_moves_nothing_keeps_the_tensors():
    lin = layer(torch.tensor([0.7]))
    before = [id(b) for b in lin.buffers()]
    lin.to("cpu")
    lin.half()
    assert [id(b) for b in lin.buffers()] == before


def test_shared_memory():
    lin = layer(torch.tensor([0.7])).share_memory()
    assert all(b.is_shared() for b in lin.buffers())


def test_a_scale_in_another_type_moves_too():
    """Refused where it is used, not where it is moved."""
    lin = layer(torch.tensor([0.7], dtype=torch.float64)).to("meta").to_empty(device="cpu")
    assert lin.act_scale.dtype == torch.float64 and lin.act_scale.device.type == "cpu"
