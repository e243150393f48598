"""Residual + RMSNorm at its borders: non-finite values in MXFP8 rows, strides and alignment, autograd."""

from __future__ import annotations

import math

import pytest
import torch

from spalmer_b200 import add_rms_norm, add_rms_norm_mxfp8
from spalmer_b200.native import mxfp8_mm_rows, mxfp8_pack_rows
from tests.test_gpu_token_norm import DEV, EPS, _inputs

pytestmark = pytest.mark.gpu


def _dequantised(values, scales):
    return values.view(torch.float8_e4m3fn).double() * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


@pytest.mark.parametrize("res", ["none", "bf16", "fp32"])
@pytest.mark.parametrize("d", [32, 768, 4128])
def test_mxfp8_rows_keep_nan(d, res):
    """A row with a NaN, and a column whose weight is one, are NaN in MXFP8 wherever they are in the BF16 rows; the
    others of a block keep their scale."""

    x, r, w = _inputs(9, d, res)
    plain = w.clone()
    x[2, 5] = math.nan
    x[4] = math.nan
    w[d - 3] = math.nan
    values, scales, _, normed = add_rms_norm_mxfp8(x, r, w, EPS, rows=True)
    got = _dequantised(values, scales)
    assert torch.isnan(normed[[2, 4]]).all() and torch.isnan(normed[:, d - 3]).all()
    assert torch.equal(torch.isnan(got), torch.isnan(normed))
    plain[d - 3] = 0.0  # as small as a block's element can be
    want = _dequantised(*add_rms_norm_mxfp8(x, r, plain, EPS)[:2])
    keep = ~torch.isnan(got)
    assert torch.equal(got[keep], want[keep])


def test_mm_rows_keep_nan():
    """A NaN row of MXFP8 values gives a NaN row of the product, and no other."""

    x, _, w = _inputs(5, 256, "none")
    x[3, 7] = math.nan
    weight = torch.randn(48, 256, device=DEV).to(torch.bfloat16)
    got = mxfp8_mm_rows(*add_rms_norm_mxfp8(x, None, w, EPS)[:2], mxfp8_pack_rows(weight))
    assert torch.isnan(got[3]).all() and torch.isfinite(got[[0, 1, 2, 4]].float()).all()


@pytest.mark.parametrize("res", ["none", "fp32"])
def test_mxfp8_rows_past_the_range(res):
    """A row whose mean square overflows FP32 is zero, as its BF16 row is; a value that is infinite there is a NaN here."""

    x, r, w = _inputs(6, 256, res)
    x[1] = 1e25
    if r is not None:
        r[4] = -1e30
    x[2, 9] = math.inf  # its own row: NaN there, zero elsewhere
    w[77] = math.inf
    values, scales, _, normed = add_rms_norm_mxfp8(x, r, w, EPS, rows=True)
    got = _dequantised(values, scales)
    assert torch.equal(torch.isnan(got), ~torch.isfinite(normed))
    zero = normed == 0
    assert zero[1].sum() == 255 and zero[2].sum() == 254 and (r is None or zero[4].sum() == 255)
    assert not got[zero].any()
    keep = torch.isfinite(normed)
    # half a step of E4M3 is 2^-4 of a value, or 2^-10 of the scale below its normal range; BF16 adds 2^-8 of a value
    step = torch.exp2(scales.double() - 127 - 10).repeat_interleave(32, -1)
    assert torch.all((got - normed.double()).abs()[keep] <= ((2.0 ** -4 + 2.0 ** -7) * normed.double().abs() + step)[keep])


@pytest.mark.parametrize("rows,d", [(7, 96), (300, 768)])
def test_fp32_rows_four_elements_apart(rows, d):
    """FP32 rows start on 16 bytes where their stride is a multiple of four elements: residual and the sum's gradient."""

    x, r, w = _inputs(rows, d, "fp32")
    g = torch.Generator(device=DEV).manual_seed(4)
    dy = torch.randn(rows, d, generator=g, device=DEV).to(torch.bfloat16)
    ds = torch.randn(rows, d, generator=g, device=DEV)

    def apart(t):
        wide = torch.full((rows, d + 4), math.nan, device=DEV)
        wide[:, :d] = t
        return wide[:, :d]

    def call(r, ds):
        ins = [t.detach().requires_grad_(True) for t in (x, r, w)]
        y, total = add_rms_norm(*ins, EPS)
        return y, total, *torch.autograd.grad((y, total), ins, (dy, ds))

    for got, want in zip(call(apart(r), apart(ds)), call(r, ds)):
        assert torch.equal(got, want)
    for got, want in zip(add_rms_norm_mxfp8(x, apart(r), w, EPS),
                         add_rms_norm_mxfp8(x, r, w, EPS)):
        assert torch.equal(got, want)


def _off(t):
    """The same values one element behind a 16-byte boundary."""

    moved = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
    moved.copy_(t)
    assert moved.data_ptr() % 16
    return moved


@pytest.mark.parametrize("res", ["none", "bf16", "fp32"])
def test_operands_off_sixteen_bytes(res):
    x, r, w = _inputs(33, 256, res)
    g = torch.Generator(device=DEV).manual_seed(6)
    dy = torch.randn(33, 256, generator=g, device=DEV).to(torch.bfloat16)

    def call(move):
        ins = [move(t).detach().requires_grad_(True) for t in (x, r, w) if t is not None]
        y, total = add_rms_norm(ins[0], ins[1] if r is not None else None, ins[-1], EPS)
        return y, total, *torch.autograd.grad(y, ins, move(dy))

    for got, want in zip(call(_off), call(lambda t: t)):
        assert torch.equal(got, want)
    rows = None if r is None else _off(r)
    for got, want in zip(add_rms_norm_mxfp8(_off(x), rows, _off(w), EPS), add_rms_norm_mxfp8(x, r, w, EPS)):
        assert torch.equal(got, want)


def test_quantised_operands_off_sixteen_bytes():
    x, _, w = _inputs(33, 256, "none")
    weight = torch.randn(48, 256, device=DEV).to(torch.bfloat16)
    values, scales, _ = add_rms_norm_mxfp8(x, None, w, EPS)
    want = mxfp8_mm_rows(values, scales, mxfp8_pack_rows(weight))
    assert torch.equal(mxfp8_mm_rows(_off(values), _off(scales), mxfp8_pack_rows(_off(weight))), want)
