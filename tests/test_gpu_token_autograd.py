"""Autograd around the token operators: what they do not differentiate raises, and what they write is known to autograd."""

from __future__ import annotations

import pytest
import torch

from spalmer_b200 import add_rms_norm, linear_attention, rotary_embed, rotary_frequencies

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _bf16(*shape, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + sum(shape))
    return torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)


def _calls():
    """name: (operator over its differentiable inputs, those inputs)"""

    pos, (freq, _) = torch.arange(20, device=DEV), rotary_frequencies(64, device=DEV)
    decay = -0.1 * torch.rand(2, 20, 2, device=DEV)
    state = torch.randn(2, 2, 64, 64, device=DEV)
    return {
        "add_rms_norm": (lambda x, w: add_rms_norm(x, None, w)[:1], (_bf16(6, 64), _bf16(64))),
        "add_rms_norm_residual": (lambda x, r, w: add_rms_norm(x, r, w), (_bf16(6, 64), _bf16(6, 64, seed=1).float(), _bf16(64))),
        "rotary_embed": (lambda q, k: rotary_embed(q, k, pos, freq), (_bf16(20, 2, 64), _bf16(20, 1, 64))),
        "linear_attention": (lambda q, k, v, a, s: linear_attention(q, k, v, a, initial_state=s, return_state=True),
                             (_bf16(2, 20, 2, 64), _bf16(2, 20, 1, 64), _bf16(2, 20, 1, 64, seed=3), decay, state)),
    }


NAMES = ("add_rms_norm", "add_rms_norm_residual", "rotary_embed", "linear_attention")


@pytest.mark.parametrize("name", NAMES)
def test_second_derivatives_raise(name):
    """A graph of the gradients gives the gradients; what is derived from it raises, even where other terms could be."""

    fn, inputs = _calls()[name]
    ins = [t.clone().requires_grad_(True) for t in inputs]
    loss = sum(y.float().square().sum() for y in fn(*ins))
    want = torch.autograd.grad(loss, ins, retain_graph=True)
    got = torch.autograd.grad(loss, ins, create_graph=True)
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    for x in got:
        with pytest.raises(NotImplementedError, match="first derivatives"):
            torch.autograd.grad(x.float().square().sum() + ins[0].float().square().sum(), ins, retain_graph=True,
                                allow_unused=True)
    # the same with constant gradients of the outputs: only the rotation, being linear, has none of its inputs in its own
    outs = fn(*ins)
    got = torch.autograd.grad(outs, ins, [torch.ones_like(y) for y in outs], create_graph=True)
    if name == "rotary_embed":
        assert not any(x.requires_grad for x in got)
    else:
        with pytest.raises(NotImplementedError, match="first derivatives"):
            (got[0].float().square().sum() + ins[0].float().square().sum()).backward()
