"""A decoder layer as a model would run it: a training step, packed prompts, and decoding.

    python -m examples.decoder_layer        (from the repository root)

Trains two layers for a few steps on random rows, then serves them: prompts of
different lengths packed into one row leave their states in a cache, and every
request decodes a few tokens from there.  Prints what decoding token by token
differs from running the whole sequences at once.
"""

from __future__ import annotations

import torch

from spalmer_b200 import (
    B200DecoderLayer,
    B200MicroExpertChannelMixer,
    LinearAttentionMixer,
    MicroExpertsConfig,
    add_rms_norm,
)


def build(d_model: int = 256, layers: int = 2) -> torch.nn.ModuleList:
    config = MicroExpertsConfig(d_model=d_model, num_experts=64, expert_inter_dim=64, shared_inter_dim=d_model,
                                active_experts=4)
    return torch.nn.ModuleList(
        B200DecoderLayer(LinearAttentionMixer(d_model, heads=4, kv_heads=2, key_dim=64, rotary_dim=32),
                         B200MicroExpertChannelMixer(config))
        for _ in range(layers)
    )


def run(layers, h, positions=None, *, cu_seqlens=None, states=None):
    """Whole sequences: (last rows, the last states of every layer, the auxiliary losses' sum)."""

    update, lasts, aux = None, [], 0.0
    for layer in layers:
        update, h, last, out = layer(update, h, positions, cu_seqlens=cu_seqlens, return_state=states is not None)
        lasts.append(last)
        aux = aux + out.auxiliary_loss.float()
    norm = layers[-1].channel_norm  # a model has a norm of its own here
    return add_rms_norm(update, h, norm.weight, norm.eps)[0], lasts, aux


def main() -> None:
    torch.manual_seed(0)
    device = torch.device("cuda")
    layers = build().to(device, torch.bfloat16)
    optimizer = torch.optim.SGD(layers.parameters(), lr=0.1)
    x, target = (torch.randn(4, 300, 256, device=device).to(torch.bfloat16) for _ in range(2))
    for step in range(3):
        rows, _, aux = run(layers, x)
        loss = (rows.float() - target.float()).square().mean() + 0.01 * aux
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
        print(f"step {step}: loss {loss.item():.4f}")

    layers.eval()
    lengths, extra = [1, 37, 128, 290], 4
    cu = torch.tensor([0, *lengths]).cumsum(0).to(device, torch.int32)
    prompts = [torch.randn(n + extra, 256, device=device).to(torch.bfloat16) for n in lengths]
    with torch.no_grad():
        packed = torch.cat([p[:n] for p, n in zip(prompts, lengths)])[None]
        positions = torch.cat([torch.arange(n, device=device) for n in lengths])[None]
        _, lasts, _ = run(layers, packed, positions, cu_seqlens=cu, states=True)
        caches = [layer.token_mixer.new_states(8) for layer in layers]
        slots = torch.tensor([5, 0, 7, 2], device=device)
        for cache, last in zip(caches, lasts):
            cache[slots] = last
        norm = layers[-1].channel_norm
        off = 0.0
        for t in range(extra):
            h = torch.stack([p[n + t] for p, n in zip(prompts, lengths)])
            at = torch.tensor([n + t for n in lengths], device=device)
            update = None
            for layer, cache in zip(layers, caches):
                update, h, _ = layer.step(update, h, at, cache, slots)
            rows = add_rms_norm(update, h, norm.weight, norm.eps)[0]
            for i, (p, n) in enumerate(zip(prompts, lengths)):
                whole, _, _ = run(layers, p[None, :n + t + 1])
                want = whole[0, -1].float()
                off = max(off, float((rows[i].float() - want).norm() / want.norm()))
    print(f"decoding differs from whole sequences by {off:.4f} (BF16 rows)")


if __name__ == "__main__":
    main()
