"""Residual addition + RMSNorm (BF16 and MXFP8 rows, gradients) and the MXFP8
GEMM on rows that are quantised already.

Tolerances.  The kernel works in FP32 and rounds once: an element of y is off
by at most half a BF16 ulp (2^-8 of it) plus FP32 roundings; the sum over a row
of d elements is taken over at most 32 elements a thread and a tree, so its
relative error is below 64 * 2^-24 = 2^-18.  Gradients: the same on the sum of
the magnitudes of the terms they are made of."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.mxfp8 import quantize_rows
from spalmer_b200 import add_rms_norm, add_rms_norm_mxfp8
from spalmer_b200.native import mx_quantize_rows, mxfp8_mm_nt, mxfp8_mm_rows, mxfp8_pack_rows
from tests.token_reference import HALF_ULP, norm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
EPS = 1e-6
FP32 = 2.0 ** -17
RES = {"none": None, "bf16": torch.bfloat16, "fp32": torch.float32}


def _inputs(rows, d, res, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + rows + d)
    x = torch.randn(rows, d, generator=g, device=DEV).to(torch.bfloat16)
    r = None if RES[res] is None else (torch.randn(rows, d, generator=g, device=DEV) * 3).to(RES[res])
    w = (1 + 0.2 * torch.randn(d, generator=g, device=DEV)).to(torch.bfloat16)
    return x, r, w


@pytest.mark.parametrize("res", RES)
@pytest.mark.parametrize("rows,d", [(0, 64), (1, 8), (3, 72), (5, 768), (37, 1032), (2, 2048), (130, 4104), (9, 8200),
                                    (3, 16384), (2500, 264)])
def test_rows(rows, d, res):
    x, r, w = _inputs(rows, d, res)
    y, total = add_rms_norm(x, r, w, EPS)
    want, summed = norm(x, r, w, EPS)
    assert y.shape == x.shape and y.dtype == torch.bfloat16
    assert torch.equal(total, summed) and total.dtype == summed.dtype
    if r is None:
        assert total is x
    assert torch.all((y.double() - want).abs() <= (HALF_ULP + FP32) * want.abs())


def test_views_and_leading_dimensions():
    """Rows of a wider tensor, three-dimensional inputs, a transposed one."""

    g = torch.Generator(device=DEV).manual_seed(1)
    wide = torch.randn(4, 9, 3 * 96, generator=g, device=DEV).to(torch.bfloat16)
    res = torch.randn(9, 4, 96, generator=g, device=DEV).transpose(0, 1)
    w = torch.ones(96, device=DEV, dtype=torch.bfloat16)
    x = wide[..., 96:192]
    y, total = add_rms_norm(x, res, w, EPS)
    want, summed = norm(x, res, w, EPS)
    assert y.shape == (4, 9, 96) and torch.equal(total, summed)
    assert torch.all((y.double() - want).abs() <= (HALF_ULP + FP32) * want.abs())
    odd = torch.randn(5 * 96 + 1, generator=g, device=DEV).to(torch.bfloat16)[1:].view(5, 96)  # 2-byte alignment
    want, _ = norm(odd, None, w, EPS)
    assert torch.all((add_rms_norm(odd, None, w, EPS)[0].double() - want).abs() <= (HALF_ULP + FP32) * want.abs())


def test_extreme_rows():
    """Zero rows stay zero (eps), huge and tiny rows keep their direction, a NaN stays in its row."""

    x = torch.zeros(4, 128, device=DEV, dtype=torch.bfloat16)
    x[1] = 1e18
    x[2] = 1e-30
    x[3, 5] = float("nan")
    w = torch.ones(128, device=DEV, dtype=torch.bfloat16)
    y, _ = add_rms_norm(x, None, w, EPS)
    want, _ = norm(x[:3], None, w, EPS)
    assert torch.all((y[:3].double() - want).abs() <= (HALF_ULP + FP32) * want.abs() + 1e-38)
    assert torch.isnan(y[3]).all()


@pytest.mark.parametrize("with_sum", [True, False])
@pytest.mark.parametrize("res", RES)
@pytest.mark.parametrize("rows,d", [(1, 8), (3, 72), (300, 768), (37, 1032), (130, 4104), (7, 8200), (3, 16384), (5000, 64)])
def test_gradients(rows, d, res, with_sum):
    if res == "none" and with_sum:
        pytest.skip("there is no sum")
    x, r, w = _inputs(rows, d, res, 7)
    g = torch.Generator(device=DEV).manual_seed(3)
    dy = torch.randn(rows, d, generator=g, device=DEV).to(torch.bfloat16)
    ds = None if r is None or not with_sum else torch.randn(rows, d, generator=g, device=DEV).to(r.dtype)
    ins = [t.requires_grad_(True) for t in (x, r, w) if t is not None]
    y, total = add_rms_norm(x, r, w, EPS)
    got = torch.autograd.grad((y, total) if ds is not None else y, ins, (dy, ds) if ds is not None else dy)
    got = dict(zip(["dx", "dres", "dw"] if r is not None else ["dx", "dw"], got))
    # the formula, in 64 bits
    h, wd = total.detach().double(), w.detach().double()
    s = 1 / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS)
    z = dy.double() * wd
    k = s.pow(3) * (z * h).mean(-1, keepdim=True)
    k_abs = s.pow(3) * (z * h).abs().mean(-1, keepdim=True)
    dh = s * z - h * k + (0 if ds is None else ds.double())
    size = (s * z).abs() + h.abs() * k_abs + (0 if ds is None else ds.double().abs())
    assert torch.all((got["dx"].double() - dh).abs() <= HALF_ULP * dh.abs() + FP32 * size)
    if r is not None:
        unit = 0.0 if r.dtype == torch.float32 else HALF_ULP
        assert got["dres"].dtype == r.dtype
        assert torch.all((got["dres"].double() - dh).abs() <= unit * dh.abs() + FP32 * size)
    terms = dy.double() * h * s
    dw = terms.sum(0)
    # a sum over rows: at most rows / 148 terms one after another, then 148 partials
    slack = 2.0 ** -24 * (rows / 100 + 200) * terms.abs().sum(0)
    assert torch.all((got["dw"].double() - dw).abs() <= HALF_ULP * dw.abs() + slack)


def test_gradient_against_differences():
    """Directional derivatives of sum(y * c), by central differences of the 64-bit form."""

    x, r, w = _inputs(6, 96, "fp32", 11)
    c = torch.randn(6, 96, device=DEV).to(torch.bfloat16)
    ins = [t.requires_grad_(True) for t in (x, r, w)]
    y, _ = add_rms_norm(x, r, w, EPS)
    grads = torch.autograd.grad(y, ins, c)
    for i, (t, grad) in enumerate(zip(ins, grads)):
        d = torch.randn(t.shape, device=DEV, dtype=torch.float64)
        step = 1e-4

        def value(sign):
            a = [u.detach().double() for u in (x, r, w)]
            a[i] = a[i] + sign * step * d
            h = a[0] + a[1]
            return float((h / torch.sqrt(h.square().mean(-1, keepdim=True) + EPS) * a[2] * c.double()).sum())

        want = (value(1) - value(-1)) / (2 * step)
        # each of the gradient's elements is rounded once (residual: FP32)
        slack = float((HALF_ULP * grad.double().abs() * d.abs()).sum()) + 1e-3
        assert abs(float((grad.double() * d).sum()) - want) <= slack


def test_backward_is_deterministic():
    x, r, w = _inputs(3000, 768, "bf16", 5)
    ins = [t.requires_grad_(True) for t in (x, r, w)]
    dy = torch.randn_like(x)

    def once():
        return torch.autograd.grad(add_rms_norm(x, r, w, EPS)[0], ins, dy)

    for a, b in zip(once(), once()):
        assert torch.equal(a, b)


@pytest.mark.parametrize("res", RES)
@pytest.mark.parametrize("rows,d", [(1, 32), (5, 768), (33, 1056), (130, 4128), (2, 16384)])
def test_mxfp8_rows(rows, d, res):
    """Values and scales against the oracle's quantiser on the 64-bit rows.  FP32
    roundings (2^-17) move a value across a rounding border of E4M3 (spaced 2^-4
    at best) in about one of 2^12 elements, and a scale across a power of two in
    about one of 2^17 blocks; a moved value is one step off."""

    x, r, w = _inputs(rows, d, res, 3)
    values, scales, total, normed = add_rms_norm_mxfp8(x, r, w, EPS, rows=True)
    want, summed = norm(x, r, w, EPS)
    assert torch.equal(total, summed)
    assert torch.equal(normed, add_rms_norm(x, r, w, EPS)[0])
    q, sb = quantize_rows(want.cpu().numpy().astype(np.float32))
    q, sb = torch.from_numpy(q), torch.from_numpy(sb)
    assert values.shape == (rows, d) and scales.shape == (rows, d // 32)
    same = (scales.cpu() == sb)
    assert float((~same).float().mean()) <= 2.0 ** -12
    got, ref = (v.view(torch.float8_e4m3fn).float() for v in (values.cpu(), q.view(torch.uint8)))
    keep = same.repeat_interleave(32, -1)
    moved = (got != ref) & keep
    assert float(moved.float().mean()) <= 2.0 ** -9
    assert torch.all((got - ref).abs()[moved] <= torch.maximum(got.abs(), ref.abs())[moved] * 2.0 ** -3 + 2.0 ** -9)


@pytest.mark.parametrize("m,n,k", [(1, 16, 128), (5, 200, 256), (130, 768, 768), (1000, 2304, 768)])
def test_mm_rows_is_mm_nt(m, n, k):
    """The same product, bit for bit, as the GEMM that quantises both operands itself."""

    g = torch.Generator(device=DEV).manual_seed(m + n)
    a = torch.randn(m, k, generator=g, device=DEV).to(torch.bfloat16)
    b = (torch.randn(n, k, generator=g, device=DEV) * 0.1).to(torch.bfloat16)
    packed = mxfp8_pack_rows(b)
    got = mxfp8_mm_rows(*mx_quantize_rows(a), packed)
    assert torch.equal(got, mxfp8_mm_nt(a, b))


def test_refusals():
    x, r, w = _inputs(4, 64, "bf16")
    with pytest.raises(ValueError, match="bfloat16"):
        add_rms_norm(x.float(), r, w)
    with pytest.raises(ValueError, match="shape"):
        add_rms_norm(x, r[:2], w)
    with pytest.raises(ValueError, match="residual"):
        add_rms_norm(x, r.half(), w)
    with pytest.raises(ValueError, match="weight"):
        add_rms_norm(x, r, w[:32])
    with pytest.raises(ValueError, match="eps"):
        add_rms_norm(x, r, w, 0.0)
    with pytest.raises(ValueError, match="block size"):
        add_rms_norm_mxfp8(x[:, :40].contiguous(), None, w[:40])
    with pytest.raises(NotImplementedError):
        add_rms_norm_mxfp8(x.clone().requires_grad_(True), r, w)
    with pytest.raises(RuntimeError, match="UNSUPPORTED"):
        add_rms_norm(x[:, :60].contiguous(), None, w[:60])
    with pytest.raises(RuntimeError, match="UNSUPPORTED"):
        wide = torch.zeros(1, 16392, device=DEV, dtype=torch.bfloat16)
        add_rms_norm(wide, None, wide[0])
    with pytest.raises(ValueError, match="128"):
        mxfp8_pack_rows(x)
