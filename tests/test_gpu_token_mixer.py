"""The token mixer and the decoder layer: the operators together, as a model runs them."""

from __future__ import annotations

import pytest
import torch
from torch.nn import functional as F

from spalmer_b200 import B200DecoderLayer, B200MicroExpertChannelMixer, LinearAttentionMixer, MicroExpertsConfig
from tests.token_reference import attention, norm, rel, rotary

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


def _layer(d=256, **kw):
    torch.manual_seed(0)
    config = MicroExpertsConfig(d_model=d, num_experts=32, expert_inter_dim=64, shared_inter_dim=d, active_experts=4)
    mixer = LinearAttentionMixer(d, heads=4, kv_heads=2, key_dim=64, rotary_dim=32, initializer_range=0.08, **kw)
    return B200DecoderLayer(mixer, B200MicroExpertChannelMixer(config)).to(DEV, torch.bfloat16).eval()


def _restated(mixer, x):
    """The mixer in 64 bits from its BF16 weights."""

    w = {n: p.detach().double() for n, p in mixer.named_parameters()}
    x = x.double()
    q, k, v = (x @ w["qkv_proj.weight"].T).split(mixer.sizes, -1)
    a = F.logsigmoid(x @ w["decay_proj.weight"].T + w["decay_proj.bias"]) / mixer.decay_span
    q, k, v = (t.unflatten(-1, (-1, mixer.key_dim)) for t in (q, k, v))
    angle = torch.arange(x.shape[1], device=x.device).double()[:, None] * mixer._frequencies
    q, k = (torch.stack([rotary(t, angle, mixer.interleaved, mixer.rotary_factor) for t in u]) for u in (q, k))
    out, last = attention(q, k, v, a, None, mixer.key_dim ** -0.5)
    return out.flatten(-2) @ w["out_proj.weight"].T, last


@pytest.mark.parametrize("interleaved", [False, True])
def test_mixer_matches_its_definition(interleaved):
    """About ten BF16 roundings lie between x and the update: 2^-8 each at most, as independent errors below 1.5%."""

    mixer = _layer(interleaved=interleaved).token_mixer
    x = torch.randn(2, 150, 256, device=DEV).to(torch.bfloat16)
    with torch.no_grad():
        got, last = mixer(x, return_state=True)
    want, want_last = _restated(mixer, x)
    assert rel(got, want) <= 0.015 and rel(last, want_last) <= 0.015


def test_layer_adds_the_residual_inside_the_norms():
    layer = _layer()
    h = torch.randn(2, 40, 256, device=DEV)  # an FP32 stream
    update = torch.randn(2, 40, 256, device=DEV).to(torch.bfloat16)
    with torch.no_grad():
        got, stream, _, out = layer(update, h)
        x, total = norm(update, h, layer.token_norm.weight, layer.token_norm.eps)
        t, _ = layer.token_mixer(x.to(torch.bfloat16))
        assert stream.dtype == torch.float32
        assert rel(stream, (total + t.float()).double()) <= 1e-4  # the norm's rounding differs in a few elements
        assert torch.equal(got, out.update)


def test_decoding_continues_prompts():
    """Packed prompts, their states in a cache, then steps: the same rows as whole sequences."""

    layer = _layer()
    lens = [1, 60, 131]
    rows = [torch.randn(n + 3, 256, device=DEV).to(torch.bfloat16) for n in lens]
    cu = torch.tensor([0, *lens]).cumsum(0).to(DEV, torch.int32)
    with torch.no_grad():
        pos = torch.cat([torch.arange(n, device=DEV) for n in lens])[None]
        _, _, last, _ = layer(None, torch.cat([r[:n] for r, n in zip(rows, lens)])[None], pos, cu_seqlens=cu, return_state=True)
        cache = layer.token_mixer.new_states(5)
        slots = torch.tensor([4, 0, 2], device=DEV)
        cache[slots] = last
        for t in range(3):
            x = torch.stack([r[n + t] for r, n in zip(rows, lens)])
            _, stream, _ = layer.step(None, x, torch.tensor(lens, device=DEV) + t, cache, slots)
            for i, (r, n) in enumerate(zip(rows, lens)):
                _, whole, _, _ = layer(None, r[None, :n + t + 1])
                # the token mixer's BF16 roundings in another order; the stream is their sum with x
                assert rel(stream[i], whole[0, -1].double()) <= 0.01


def test_training_reaches_every_parameter():
    layer = _layer().train()
    x = torch.randn(2, 130, 256, device=DEV).to(torch.bfloat16).requires_grad_(True)
    update, h, _, out = layer(None, x)
    ((update.float() + h.float()).square().mean() + 0.01 * out.auxiliary_loss.float()).backward()
    assert x.grad is not None and torch.isfinite(x.grad.float()).all() and x.grad.any()
    for name, p in layer.named_parameters():
        assert p.grad is not None and torch.isfinite(p.grad.float()).all(), name
        assert p.grad.any(), name


def test_mxfp8_projection():
    """E4M3 operands carry 2^-4 of an element at most: some 3% of the projection in the mean."""

    layer = _layer()
    x = torch.randn(3, 70, 256, device=DEV).to(torch.bfloat16)
    with torch.no_grad():
        want = layer(None, x)[1]
        t = want.double() - x.double()
        layer.pack_mxfp8()
        got = layer(None, x)[1]
        assert not torch.equal(got, want)
        assert float((got.double() - want.double()).norm() / t.norm()) <= 0.12
        layer.pack_mxfp8(False)
        assert torch.equal(layer(None, x)[1], want)


def test_refusals():
    layer = _layer()
    with pytest.raises(ValueError, match="batch, seq"):
        layer.token_mixer(torch.zeros(3, 256, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="batch"):
        layer.token_mixer.step(torch.zeros(3, 1, 256, device=DEV, dtype=torch.bfloat16), None, None)
    with pytest.raises(ValueError, match="d_model"):
        B200DecoderLayer(LinearAttentionMixer(128, 2), layer.channel_mixer)
