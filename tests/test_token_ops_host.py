"""The token operators' host side: frequency tables, refusals and sizes, without a GPU."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from spalmer_b200 import (
    LinearAttentionMixer,
    _lib,
    add_rms_norm,
    add_rms_norm_mxfp8,
    linear_attention,
    linear_attention_step,
    rotary_embed,
    rotary_frequencies,
)


def test_rotary_frequencies():
    freq, factor = rotary_frequencies(64)
    assert freq.dtype == torch.float64 and freq.shape == (32,) and factor == 1.0
    assert freq[0] == 1.0 and math.isclose(float(freq[-1]), 10000.0 ** (-62 / 64))
    linear, _ = rotary_frequencies(64, scaling="linear", factor=8.0)
    assert torch.allclose(linear, freq / 8, rtol=1e-15)
    ntk, _ = rotary_frequencies(64, scaling="ntk", factor=8.0)
    assert ntk[0] == 1.0  # the fastest pair is kept, the slowest divided by the factor
    assert math.isclose(float(ntk[-1]), float(freq[-1]) / 8, rel_tol=1e-12)
    yarn, factor = rotary_frequencies(128, scaling="yarn", factor=16.0, original_length=4096)
    base, _ = rotary_frequencies(128)
    turns = 4096 * base / (2 * math.pi)
    assert torch.equal(yarn[turns > 33], base[turns > 33])
    assert torch.allclose(yarn[turns < 0.9], base[turns < 0.9] / 16, rtol=1e-15)
    assert torch.all(yarn <= base) and torch.all(yarn >= base / 16)
    assert math.isclose(factor, 0.1 * math.log(16) + 1)
    assert rotary_frequencies(0)[0].shape == (0,)
    for bad in (dict(rotary_dim=7), dict(rotary_dim=8, scaling="other"), dict(rotary_dim=8, factor=0.5),
                dict(rotary_dim=2, scaling="ntk"), dict(rotary_dim=8, base=1.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad)


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 32, dtype=torch.bfloat16), torch.ones(32, dtype=torch.bfloat16)
    q = torch.zeros(1, 2, 1, 32, dtype=torch.bfloat16)
    g = torch.zeros(1, 2, 1)
    for call in (lambda: add_rms_norm(x, None, w), lambda: add_rms_norm_mxfp8(x, None, w),
                 lambda: rotary_embed(q, q, torch.arange(2), rotary_frequencies(32)[0]),
                 lambda: linear_attention(q, q, q, g),
                 lambda: linear_attention_step(q[0], q[0], q[0], g[0], torch.zeros(2, 1, 32, 32))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_mixer_construction():
    mixer = LinearAttentionMixer(96, 6, kv_heads=2, key_dim=32, value_dim=64)
    assert mixer.qkv_proj.weight.shape == (6 * 32 + 2 * 32 + 2 * 64, 96)
    assert mixer.out_proj.weight.shape == (96, 6 * 64)
    assert mixer.to(torch.bfloat16)._frequencies.dtype == torch.float64
    assert set(mixer.state_dict()) == {"qkv_proj.weight", "decay_proj.weight", "decay_proj.bias", "out_proj.weight"}
    assert mixer.new_states(3).shape == (3, 6, 32, 64)
    for bad in (dict(heads=3, kv_heads=2), dict(heads=2, rotary_dim=128), dict(heads=2, decay_span=0.0)):
        with pytest.raises(ValueError):
            LinearAttentionMixer(96, **bad)


def test_null_pointers_and_bad_shapes_are_rejected():
    lib = _lib.load()
    assert lib.spx_add_rmsnorm_rows(None, 64, None, 0, 0, None, 1e-6, 4, 64, None, None, None, None, None) == -1
    assert lib.spx_add_rmsnorm_rows(None, 64, None, 0, 0, None, 0.0, 0, 64, None, None, None, None, None) == -1
    assert lib.spx_add_rmsnorm_rows(None, 60, None, 0, 0, None, 1e-6, 4, 60, None, None, None, None, None) == -2
    assert lib.spx_add_rmsnorm_rows(None, 64, None, 0, 0, None, 1e-6, 0, 64, None, None, None, None, None) == 0
    assert lib.spx_add_rmsnorm_backward(None, 64, 0, None, 1e-6, None, 64, None, 0, 4, 64, None, None, None, None, 0,
                                        None) == -1
    heads = _lib.Heads(None, 0, 64, 64)
    assert lib.spx_rotary(heads, 2, heads, 2, 4, 64, 32, None, 1, 4, None, 1.0, 0, 0, None, None, None) == -1
    assert lib.spx_rotary(heads, 2, heads, 2, 4, 64, 40, None, 1, 4, None, 1.0, 0, 0, None, None, None) == -1
    assert lib.spx_rotary(heads, 2, heads, 2, 4, 8192, 32, None, 1, 4, None, 1.0, 0, 0, None, None, None) == -2
    g = _lib.Decays(None, 0, 0, 0)
    dims = _lib.LinAttnDims(2, 300, 4, 2, 64, 64, 0, 1, 0.125)
    args = (heads, heads, heads, g, None, None, None, None, None, 0, None, None)
    assert lib.spx_linear_attention(dims, *args) == -1
    for field, value, rc in (("heads", 3, -1), ("key_dim", 60, -2), ("value_dim", 136, -2), ("scale", 0.0, -1),
                             ("batch", -1, -1), ("scale", float("nan"), -1), ("kv_heads", 0, -1)):
        bad = _lib.LinAttnDims(2, 300, 4, 2, 64, 64, 0, 1, 0.125)
        setattr(bad, field, value)
        assert lib.spx_linear_attention(bad, *args) == rc, field
        assert lib.spx_linear_attention_workspace(bad) == 0
    packed = _lib.LinAttnDims(2, 300, 4, 2, 64, 64, 1, 1, 0.125)
    assert lib.spx_linear_attention(packed, *args) == -1  # no offsets
    assert lib.spx_linear_attention_step(heads, heads, heads, g, 1, 3, 4, 2, 64, 64, 0.125, None, 2, None, None, None) == -1
    assert lib.spx_mxfp8_mm_rows(None, None, None, None, 4, 16, 128, None, None, None) == -1
    assert lib.spx_mxfp8_mm_rows(None, None, None, None, 4, 16, 96, None, None, None) == -2
    sizes = ctypes.c_size_t(), ctypes.c_size_t()
    assert lib.spx_mxfp8_packed_sizes(200, 256, *sizes) == 0
    assert sizes[0].value == 200 * 256 and sizes[1].value % 512 == 0


def test_workspace_sizes():
    lib = _lib.load()
    many = _lib.LinAttnDims(64, 1024, 12, 12, 64, 64, 0, 1, 0.125)
    assert lib.spx_linear_attention_workspace(many) == 0  # enough heads: no segments
    long = _lib.LinAttnDims(1, 65536, 2, 2, 128, 128, 0, 1, 0.125)
    assert lib.spx_linear_attention_workspace(long) > 0
    plain = lib.spx_linear_attention_backward_workspace(many)
    shared = _lib.LinAttnDims(64, 1024, 12, 4, 64, 64, 0, 1, 0.125)
    n = 64 * 1024 * 12
    # shared heads keep their FP32 gradients per query head
    assert lib.spx_linear_attention_backward_workspace(shared) >= plain + n * 64 * 4 * 2
    assert plain >= 2 * n * 4 + 64 * 12 * 64 * 64 * 4
    assert lib.spx_add_rmsnorm_backward_workspace(1000, 768) % (768 * 4) == 0
    assert lib.spx_add_rmsnorm_backward_workspace(0, 768) == 0
