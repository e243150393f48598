"""The decoder layer's MXFP8 projection follows its weight."""

from __future__ import annotations

import copy

import pytest
import torch
from torch import nn

from tests.test_gpu_token_mixer import DEV, _layer

pytestmark = pytest.mark.gpu


def _train_step(layer):
    x = torch.randn(2, 20, 256, device=DEV).to(torch.bfloat16)
    layer.train()
    optimizer = torch.optim.SGD(layer.parameters(), lr=0.5)
    update, h, _, _ = layer(None, x)
    (update.float() + h.float()).square().mean().backward()
    optimizer.step()
    layer.eval()


CHANGES = {
    "in_place": lambda layer: layer.token_mixer.qkv_proj.weight.neg_(),
    "optimiser": _train_step,
    "load_state_dict": lambda layer: layer.load_state_dict(
        {k: -v if v.is_floating_point() else v for k, v in layer.state_dict().items()}),
    "new_parameter": lambda layer: setattr(layer.token_mixer.qkv_proj, "weight",
                                           nn.Parameter(-layer.token_mixer.qkv_proj.weight.detach())),
    "moved": lambda layer: layer.to("cpu").to(DEV),
    "nothing": lambda layer: None,
}


@pytest.mark.parametrize("change", CHANGES)
def test_packed_projection_follows_its_weight(change):
    layer = _layer()
    x = torch.randn(3, 70, 256, device=DEV).to(torch.bfloat16)
    with torch.no_grad():
        layer.pack_mxfp8()
        before = layer(None, x)[1]
    with torch.set_grad_enabled(change == "optimiser"):
        CHANGES[change](layer)
    with torch.no_grad():
        got = layer(None, x)[1]
        fresh = copy.deepcopy(layer)
        fresh.pack_mxfp8()
        assert torch.equal(got, fresh(None, x)[1])
        assert torch.equal(got, before) == (change in ("moved", "nothing"))
        layer.pack_mxfp8(False)
        assert not torch.equal(layer(None, x)[1], got)


def test_unchanged_weight_is_packed_once():
    layer = _layer()
    x = torch.randn(1, 9, 256, device=DEV).to(torch.bfloat16)
    with torch.no_grad():
        layer.pack_mxfp8()
        first = layer._packed_projection()[0]
        layer(None, x)
        assert layer._packed_projection()[0] is first
