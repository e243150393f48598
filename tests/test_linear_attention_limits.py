"""Sizes that 32-bit coordinates cannot hold are refused before anything is launched."""

from __future__ import annotations

import ctypes

import pytest

from spalmer_b200 import _lib

UNSUPPORTED = -2


@pytest.mark.parametrize("batch,heads,value_dim", [(16386, 65528, 128), (1 << 40, 1, 64), (4, 65536, 64)])
def test_too_many_sequences_and_heads(batch, heads, value_dim):
    """Lanes (a sequence, head and 64 value columns each) are walked in steps of the SMs: one past the last has to be an int.
    The pointers are never used."""

    buffer = ctypes.create_string_buffer(64)
    at = (ctypes.addressof(buffer) + 15) // 16 * 16
    heads_of = _lib.Heads(at, 0, 8 * heads, 8)
    dims = _lib.LinAttnDims(batch, 1, heads, heads, 8, value_dim, 1, 1, 1.0)
    args = (heads_of, heads_of, heads_of, _lib.Decays(at, 0, heads, 1), at, None, at, None, None, 0, None, None)
    assert _lib.load().spx_linear_attention(dims, *args) == UNSUPPORTED
