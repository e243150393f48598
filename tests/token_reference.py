"""Plain 64-bit forms of the token operators, by their definitions."""

from __future__ import annotations

import torch
from torch import Tensor

HALF_ULP = 2.0 ** -8  # the largest relative error of one rounding to BF16
MEAN_ULP = HALF_ULP / 3 ** 0.5  # and an upper bound of its root mean square


def norm(hidden: Tensor, residual: Tensor | None, weight: Tensor, eps: float) -> tuple[Tensor, Tensor]:
    """(normed, summed): the norm is that of the sum as it is stored."""

    summed = hidden if residual is None else (hidden.float() + residual.float()).to(residual.dtype)
    h = summed.double()
    return h / torch.sqrt(h.square().mean(-1, keepdim=True) + eps) * weight.double(), summed


def rotary(x: Tensor, angle: Tensor, interleaved: bool, factor: float) -> Tensor:
    """x [tokens, heads, d], angle [tokens, pairs]."""

    pairs = angle.shape[-1]
    y = x.double().clone()
    a, b = (slice(0, 2 * pairs, 2), slice(1, 2 * pairs, 2)) if interleaved else (slice(0, pairs), slice(pairs, 2 * pairs))
    u, v = x.double()[..., a], x.double()[..., b]
    c, s = factor * angle.cos()[:, None], factor * angle.sin()[:, None]
    y[..., a], y[..., b] = u * c - v * s, v * c + u * s
    return y


def attention(q: Tensor, k: Tensor, v: Tensor, g: Tensor, state: Tensor | None, scale: float,
              cu: list[int] | None = None) -> tuple[Tensor, Tensor]:
    """Token by token; 64-bit inputs, differentiable."""

    if cu is not None:
        outs, lasts = [], []
        for i, (lo, hi) in enumerate(zip(cu, cu[1:])):
            o, s = attention(q[:, lo:hi], k[:, lo:hi], v[:, lo:hi], g[:, lo:hi], None if state is None else state[i:i + 1],
                             scale)
            outs.append(o)
            lasts.append(s)
        return torch.cat(outs, 1), torch.cat(lasts, 0)
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    group = H // k.shape[2]
    k, v = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
    S = torch.zeros(B, H, dk, dv, dtype=q.dtype, device=q.device) if state is None else state
    out = []
    for t in range(T):
        S = torch.exp(g[:, t])[..., None, None] * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        out.append(scale * (q[:, t, :, None] @ S)[:, :, 0])
    return (torch.stack(out, 1) if out else q.new_zeros(B, 0, H, dv)), S


def rel(got: Tensor, want: Tensor) -> float:
    return float((got.detach().double() - want.detach()).norm() / want.detach().norm().clamp(min=1e-300))
