"""Autograd around the token operators: what they do not differentiate raises, and what they write is known to autograd."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

from spalmer_b200 import (
    add_rms_norm,
    add_rms_norm_mxfp8,
    linear_attention,
    linear_attention_step,
    rotary_embed,
    rotary_frequencies,
)

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


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("name", [*NAMES, "add_rms_norm_mxfp8", "linear_attention_step"])
def test_tangents_are_refused(name, requires_grad):
    """Whichever input has one; a call without one works beside them."""

    calls = _calls() | {
        "add_rms_norm_mxfp8": (add_rms_norm_mxfp8, (_bf16(6, 64), _bf16(6, 64, seed=1), _bf16(64))),
        "linear_attention_step": (linear_attention_step, (_bf16(2, 2, 64), _bf16(2, 1, 64), _bf16(2, 1, 64),
                                                          -torch.rand(2, 2, device=DEV),
                                                          torch.zeros(2, 2, 64, 64, device=DEV))),
    }
    fn, inputs = calls[name]
    if requires_grad and name not in NAMES:
        pytest.skip("forward only")
    for i in range(len(inputs)):
        with forward_ad.dual_level():
            fn(*inputs)
            ins = [t.clone().requires_grad_(requires_grad) for t in inputs]
            ins[i] = forward_ad.make_dual(ins[i], torch.ones_like(ins[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(*ins)


def test_a_step_is_a_change_of_its_state():
    """A state kept for a backward pass and then stepped is noticed; one that only inference has seen may be stepped."""

    _, (q, k, v, a, state) = _calls()["linear_attention"]
    q = q.clone().requires_grad_(True)
    out, _ = linear_attention(q, k, v, a, initial_state=state)
    before = state._version
    with torch.no_grad():
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], a[:, 0], state)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.float().sum().backward()
    with torch.inference_mode():
        cache = torch.zeros_like(state)
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], a[:, 0], cache)
        assert cache.any()
