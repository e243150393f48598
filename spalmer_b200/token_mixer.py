"""A token mixer of linear attention, and a whole block around the channel mixer.

``LinearAttentionMixer`` runs the token operators together: one projection to
queries, keys, values and decays, rotary positions, linear attention with a
decay per head, and the output projection.  ``B200DecoderLayer`` puts it in
front of ``B200MicroExpertChannelMixer``, with the residual stream added inside
the two norms (``add_rms_norm``).  Both train; both decode token by token from a
cache of states; in evaluation the layer's first projection can run from MXFP8
rows (``pack_mxfp8``).
"""

from __future__ import annotations

import torch
from torch import Tensor, nn
from torch.nn import functional as F

from spalmer_b200.experts import B200MicroExpertChannelMixer, ChannelMixerOutput, RMSNorm
from spalmer_b200.native import mxfp8_mm_rows, mxfp8_pack_rows
from spalmer_b200.token_ops import (
    add_rms_norm,
    add_rms_norm_mxfp8,
    linear_attention,
    linear_attention_step,
    rotary_embed,
    rotary_frequencies,
)


class LinearAttentionMixer(nn.Module):
    """Linear attention over normalised hidden rows ``[batch, seq, d_model]``.

    A head forgets by ``exp(log_sigmoid(x w + b) / decay_span)`` a token: with a
    zero input and ``b = 0`` half of its state is left after ``decay_span`` tokens.
    ``rotary_dim`` elements of each key-dimension head carry positions (0: none).
    """

    def __init__(self, d_model: int, heads: int, *, kv_heads: int | None = None, key_dim: int = 64,
                 value_dim: int | None = None, rotary_dim: int | None = None, rotary_base: float = 10000.0,
                 rotary_scaling: str | None = None, rotary_factor: float = 1.0, interleaved: bool = False,
                 decay_span: float = 16.0, initializer_range: float = 0.02) -> None:
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        value_dim = key_dim if value_dim is None else value_dim
        rotary_dim = key_dim if rotary_dim is None else rotary_dim
        if d_model < 1 or heads < 1 or kv_heads < 1 or heads % kv_heads:
            raise ValueError("d_model, heads and kv_heads must be positive, heads a multiple of kv_heads")
        if rotary_dim > key_dim or decay_span <= 0:
            raise ValueError("rotary_dim must not exceed key_dim and decay_span must be positive")
        self.d_model, self.heads, self.kv_heads = d_model, heads, kv_heads
        self.key_dim, self.value_dim, self.interleaved, self.decay_span = key_dim, value_dim, interleaved, decay_span
        self.sizes = (heads * key_dim, kv_heads * key_dim, kv_heads * value_dim)
        self.qkv_proj = nn.Linear(d_model, sum(self.sizes), bias=False)
        self.decay_proj = nn.Linear(d_model, heads, bias=True)
        self.out_proj = nn.Linear(heads * value_dim, d_model, bias=False)
        for proj in (self.qkv_proj, self.decay_proj, self.out_proj):
            nn.init.normal_(proj.weight, std=initializer_range)
        nn.init.zeros_(self.decay_proj.bias)
        freq, self.rotary_factor = rotary_frequencies(rotary_dim, rotary_base, scaling=rotary_scaling,
                                                      factor=rotary_factor)
        self._frequencies = freq  # FP64: not a buffer, so that .to(bfloat16) leaves it alone

    def _apply(self, fn, recurse: bool = True):
        super()._apply(fn, recurse)
        self._frequencies = self._frequencies.to(self.out_proj.weight.device)
        return self

    def new_states(self, slots: int) -> Tensor:
        """A cache of ``slots`` empty states (FP32 [slots, heads, key_dim, value_dim])."""

        return torch.zeros(slots, self.heads, self.key_dim, self.value_dim, dtype=torch.float32,
                           device=self.out_proj.weight.device)

    def _project(self, x: Tensor, qkv: Tensor | None) -> tuple[Tensor, Tensor, Tensor, Tensor]:
        """q, k, v as views of one projection [..., heads, dim], and the log decays [..., heads]."""

        if qkv is None:
            qkv = self.qkv_proj(x)
        lead = qkv.shape[:-1]
        q, k, v = qkv.split(self.sizes, dim=-1)
        decay = F.logsigmoid(self.decay_proj(x)) / self.decay_span
        return (q.unflatten(-1, (self.heads, self.key_dim)), k.unflatten(-1, (self.kv_heads, self.key_dim)),
                v.unflatten(-1, (self.kv_heads, self.value_dim)), decay.reshape(*lead, self.heads))

    def forward(self, x: Tensor, positions: Tensor | None = None, *, initial_state: Tensor | None = None,
                cu_seqlens: Tensor | None = None, return_state: bool = False,
                qkv: Tensor | None = None) -> tuple[Tensor, Tensor | None]:
        """``(update, last_state or None)`` of ``x`` [batch, seq, d_model].

        ``positions``: [seq] or [batch, seq] integers (default 0, 1, ...; packed
        sequences pass their own); ``cu_seqlens``, ``initial_state`` and
        ``return_state`` as in ``linear_attention``; ``qkv``: the projection, where
        the caller has computed it.
        """

        if x.ndim != 3 or x.shape[-1] != self.d_model:
            raise ValueError(f"x must be [batch, seq, {self.d_model}]")
        if positions is None:
            positions = torch.arange(x.shape[1], device=x.device)
        q, k, v, decay = self._project(x, qkv)
        if self._frequencies.numel():
            q, k = rotary_embed(q, k, positions, self._frequencies, interleaved=self.interleaved,
                                factor=self.rotary_factor)
        out, last = linear_attention(q, k, v, decay, initial_state=initial_state, cu_seqlens=cu_seqlens,
                                     return_state=return_state)
        return self.out_proj(out.flatten(-2)), last

    def step(self, x: Tensor, positions: Tensor, state: Tensor, slots: Tensor | None = None, *,
             qkv: Tensor | None = None) -> Tensor:
        """The update of one token a request, ``x`` [batch, d_model], states updated in place."""

        if x.ndim != 2 or x.shape[-1] != self.d_model:
            raise ValueError(f"x must be [batch, {self.d_model}]")
        q, k, v, decay = self._project(x, qkv)
        if self._frequencies.numel():
            q, k = rotary_embed(q, k, positions, self._frequencies, interleaved=self.interleaved,
                                factor=self.rotary_factor)
        return self.out_proj(linear_attention_step(q, k, v, decay, state, slots=slots).flatten(-2))


class B200DecoderLayer(nn.Module):
    """Token mixer and micro-expert channel mixer around one residual stream.

    The stream ``h`` is kept apart from the update that the layer before left
    (``update`` may be None at the first layer), and every addition happens
    inside the norm that needs its sum:

        x, h = add_rms_norm(update, h, token_norm);    t = token_mixer(x)
        y, h = add_rms_norm(t, h, channel_norm);       update = channel_mixer(y).update

    ``forward`` and ``step`` return ``(update, h, ...)`` for the next layer; after
    the last one the final norm adds them once more.  ``h`` is BF16 or FP32.
    """

    def __init__(self, token_mixer: LinearAttentionMixer, channel_mixer: B200MicroExpertChannelMixer, *,
                 eps: float = 1e-6) -> None:
        super().__init__()
        if token_mixer.d_model != channel_mixer.config.d_model:
            raise ValueError("both mixers must have one d_model")
        self.token_mixer, self.channel_mixer = token_mixer, channel_mixer
        self.token_norm, self.channel_norm = RMSNorm(token_mixer.d_model, eps), RMSNorm(token_mixer.d_model, eps)
        object.__setattr__(self, "_mxfp8", None)

    def pack_mxfp8(self, on: bool = True) -> None:
        """Serve the first projection in MXFP8 (d_model a multiple of 128): its weight is packed
        now, and again when it has changed, and while gradients are off the first norm writes
        MXFP8 rows for it."""

        object.__setattr__(self, "_mxfp8", None)
        if on:
            self._packed_projection()

    def _packed_projection(self) -> tuple[Tensor, Tensor, tuple[int, int]]:
        """The first projection's weight in MXFP8, packed anew where the weight is not the one packed before."""

        weight = self.token_mixer.qkv_proj.weight.detach()
        key = (weight.device, weight.dtype, weight.data_ptr(), weight._version)
        if self._mxfp8 is None or self._mxfp8[0] != key:
            # the weight is kept with it, so that no other one can come to lie at its address
            object.__setattr__(self, "_mxfp8", (key, weight, mxfp8_pack_rows(weight.to(torch.bfloat16))))
        return self._mxfp8[2]

    def _enter(self, update: Tensor | None, h: Tensor) -> tuple[Tensor, Tensor | None, Tensor]:
        """(normalised rows, the projection in MXFP8 or None, the stream)."""

        norm = self.token_norm
        first = h.to(torch.bfloat16) if update is None else update  # the stream itself, in BF16
        residual = None if update is None else h
        if self._mxfp8 is None or torch.is_grad_enabled():
            x, total = add_rms_norm(first, residual, norm.weight, norm.eps)
            return x, None, h if update is None else total
        values, scales, total, x = add_rms_norm_mxfp8(first, residual, norm.weight, norm.eps, rows=True)
        return x, mxfp8_mm_rows(values, scales, self._packed_projection()), h if update is None else total

    def _leave(self, t: Tensor, h: Tensor) -> tuple[Tensor, Tensor, ChannelMixerOutput]:
        y, h = add_rms_norm(t, h, self.channel_norm.weight, self.channel_norm.eps)
        out = self.channel_mixer(y if y.ndim == 3 else y[:, None])
        return out.update.reshape(y.shape), h, out

    def forward(self, update: Tensor | None, h: Tensor, positions: Tensor | None = None, *,
                initial_state: Tensor | None = None, cu_seqlens: Tensor | None = None,
                return_state: bool = False) -> tuple[Tensor, Tensor, Tensor | None, ChannelMixerOutput]:
        """``(update, h, last_state or None, channel output)`` of ``[batch, seq, d_model]`` rows."""

        x, qkv, h = self._enter(update, h)
        t, last = self.token_mixer(x, positions, initial_state=initial_state, cu_seqlens=cu_seqlens,
                                   return_state=return_state, qkv=qkv)
        update, h, out = self._leave(t, h)
        return update, h, last, out

    def step(self, update: Tensor | None, h: Tensor, positions: Tensor, state: Tensor,
             slots: Tensor | None = None) -> tuple[Tensor, Tensor, ChannelMixerOutput]:
        """One token a request (``[batch, d_model]`` rows): ``(update, h, channel output)``."""

        x, qkv, h = self._enter(update, h)
        update, h, out = self._leave(self.token_mixer.step(x, positions, state, slots, qkv=qkv), h)
        return update, h, out


__all__ = ["B200DecoderLayer", "LinearAttentionMixer"]
