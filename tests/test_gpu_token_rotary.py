"""Rotary positions against the 64-bit rotation.

Tolerance: one rounding to BF16 (2^-8 of the result) plus, on the magnitudes
of the two elements of a pair, the sine's and cosine's error: 2^-21 of the fast
functions, 2^-24 each of the angle's reduction to FP32 (times 2 pi) and of the
products -- together below 2^-19."""

from __future__ import annotations

import pytest
import torch

from spalmer_b200 import rotary_embed, rotary_frequencies
from tests.token_reference import HALF_ULP, rotary

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
TRIG = 2.0 ** -19


def _check(got, x, pos, freq, interleaved, factor):
    angle = pos.double()[:, None] * freq
    want = rotary(x, angle, interleaved, factor)
    pairs = freq.shape[0]
    size = torch.zeros_like(want)
    if pairs:
        size[..., :2 * pairs] = factor * x.double()[..., :2 * pairs].abs().amax(-1, keepdim=True) * 2
    assert torch.all((got.double() - want).abs() <= HALF_ULP * want.abs() + TRIG * size)
    assert torch.equal(got[..., 2 * pairs:], x[..., 2 * pairs:])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("tokens,heads,kv,d,rot", [(1, 1, 1, 16, 16), (3, 2, 1, 64, 32), (131, 12, 12, 64, 64),
                                                   (5, 3, 3, 40, 20), (17, 4, 2, 80, 40), (2, 1, 1, 6, 4), (9, 2, 2, 128, 0),
                                                   (1000, 5, 1, 256, 128), (4, 40, 8, 128, 128), (2, 1, 1, 4096, 4096)])
def test_layouts(tokens, heads, kv, d, rot, interleaved):
    g = torch.Generator(device=DEV).manual_seed(tokens + d)
    q = torch.randn(tokens, heads, d, generator=g, device=DEV).to(torch.bfloat16)
    k = torch.randn(tokens, kv, d, generator=g, device=DEV).to(torch.bfloat16)
    pos = torch.randint(0, 5000, (tokens,), generator=g, device=DEV)
    freq, _ = rotary_frequencies(rot, device=DEV)
    a, b = rotary_embed(q, k, pos, freq, interleaved=interleaved, factor=1.25)
    _check(a, q, pos, freq, interleaved, 1.25)
    _check(b, k, pos, freq, interleaved, 1.25)
    only, none = rotary_embed(q, None, pos.int(), freq, interleaved=interleaved, factor=1.25)
    assert none is None and torch.equal(only, a)


@pytest.mark.parametrize("interleaved", [False, True])
def test_views_of_a_fused_projection(interleaved):
    g = torch.Generator(device=DEV).manual_seed(2)
    qkv = torch.randn(2, 50, 10 * 64 + 8, generator=g, device=DEV).to(torch.bfloat16)
    q, k = qkv[..., :6 * 64].unflatten(-1, (6, 64)), qkv[..., 6 * 64 + 8:8 * 64 + 8].unflatten(-1, (2, 64))
    odd = qkv[..., 3:3 + 64].unflatten(-1, (1, 64))  # 2-byte alignment: element by element
    freq, _ = rotary_frequencies(64, device=DEV)
    pos = torch.arange(50, device=DEV)
    both = pos.repeat(2)
    for x in (q, k, odd):
        got, _ = rotary_embed(x, None, pos, freq, interleaved=interleaved)
        assert got.shape == x.shape and got.is_contiguous()
        _check(got.reshape(100, -1, 64), x.reshape(100, -1, 64), both, freq, interleaved, 1.0)
        again, _ = rotary_embed(x, None, both.view(2, 50), freq, interleaved=interleaved)
        assert torch.equal(got, again)


def test_far_and_negative_positions():
    """Positions past 2^31: the angle is reduced in 64 bits (and the reference in whole turns)."""

    q = torch.randn(5, 2, 32, device=DEV).to(torch.bfloat16)
    pos = torch.tensor([0, -7, 999_983, 2 ** 31 + 11, 2 ** 33 + 1], device=DEV)
    freq, _ = rotary_frequencies(32, device=DEV)
    got, _ = rotary_embed(q, None, pos, freq)
    # positions times frequencies lose 2^-53 of up to 2^33: below 2^-19 still
    _check(got, q, pos, freq, False, 1.0)


@pytest.mark.parametrize("interleaved", [False, True])
def test_gradients(interleaved):
    g = torch.Generator(device=DEV).manual_seed(4)
    q = torch.randn(70, 4, 72, generator=g, device=DEV).to(torch.bfloat16).requires_grad_(True)
    k = torch.randn(70, 2, 72, generator=g, device=DEV).to(torch.bfloat16).requires_grad_(True)
    pos = torch.randint(0, 10000, (70,), generator=g, device=DEV)
    freq, _ = rotary_frequencies(32, device=DEV)
    a, b = rotary_embed(q, k, pos, freq, interleaved=interleaved, factor=0.5)
    da, db = torch.randn(a.shape, device=DEV).to(a), torch.randn(b.shape, device=DEV).to(b)
    for got, dy in zip(torch.autograd.grad((a, b), (q, k), (da, db)), (da, db)):
        _check(got, dy, -pos, freq, interleaved, 0.5)
    # the map is linear: <R x, y> = <x, R^T y>, each side rounded once an element
    lhs = (a.detach().double() * da.double()).sum()
    rhs = (q.detach().double() * rotary_embed(da, None, -pos, freq, interleaved=interleaved, factor=0.5)[0].double()).sum()
    slack = HALF_ULP * float((a.detach().double() * da.double()).abs().sum() + (q.detach().double() * da.double()).abs().sum())
    assert abs(float(lhs - rhs)) <= slack
    # only one of the two takes part in the loss
    a, b = rotary_embed(q, k, pos, freq, interleaved=interleaved)
    dq, dk = torch.autograd.grad(a, (q, k), da, allow_unused=True)
    assert dq is not None and (dk is None or not dk.any())


def test_empty_and_refusals():
    freq, _ = rotary_frequencies(32, device=DEV)
    q = torch.zeros(0, 2, 32, device=DEV, dtype=torch.bfloat16)
    assert rotary_embed(q, q, torch.zeros(0, device=DEV, dtype=torch.int64), freq)[0].shape == (0, 2, 32)
    q = torch.zeros(4, 2, 32, device=DEV, dtype=torch.bfloat16)
    pos = torch.arange(4, device=DEV)
    with pytest.raises(ValueError, match="bfloat16"):
        rotary_embed(q.float(), None, pos, freq)
    with pytest.raises(ValueError, match="positions"):
        rotary_embed(q, None, pos.float(), freq)
    with pytest.raises(ValueError, match="positions"):
        rotary_embed(q, None, pos[:3], freq)
    with pytest.raises(ValueError, match="frequencies"):
        rotary_embed(q, None, pos, freq.float())
    with pytest.raises(ValueError, match="frequencies"):
        rotary_embed(q[..., :24].contiguous(), None, pos, freq)
    with pytest.raises(ValueError, match="q's tokens"):
        rotary_embed(q, q[:2], pos, freq)
    with pytest.raises(ValueError, match="on cpu|CUDA"):
        rotary_embed(q, None, pos.cpu(), freq)
