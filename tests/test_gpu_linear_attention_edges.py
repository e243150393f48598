"""Linear attention at its borders: neighbours in a packed row, rows of no sequence, views, autograd."""

from __future__ import annotations

import math

import pytest
import torch

from spalmer_b200 import _lib, linear_attention, linear_attention_status
from tests.test_gpu_linear_attention import DEV, _inputs

pytestmark = pytest.mark.gpu


def _tails(kind):
    """Packed lengths whose tails end all over a chunk: many short ones, or a few long enough to be cut into segments."""

    if kind == "segments":
        return [4000, 70, 9000, 33, 7001]
    g = torch.Generator().manual_seed(17)
    sizes = (1, 5, 37, 64, 100, 129, 200)
    return [sizes[i] for i in torch.randint(len(sizes), (121,), generator=g).tolist()]


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("kind,H,kv,dk,dv", [("short", 4, 4, 64, 64), ("short", 4, 2, 128, 128), ("short", 2, 1, 64, 120),
                                             ("segments", 1, 1, 64, 64), ("segments", 1, 1, 128, 72)])
def test_non_finite_neighbours_at_every_tail(kind, H, kv, dk, dv, bad):
    """Every second sequence holds NaN or infinities; the ones between them come out, and train, with the same bits as
    among finite neighbours."""

    lens = _tails(kind)
    cu = [0] + torch.tensor(lens).cumsum(0).tolist()
    cut = torch.tensor(cu, device=DEV, dtype=torch.int32)
    if kind == "segments":
        dims = _lib.LinAttnDims(len(lens), cu[-1], H, kv, dk, dv, 1, 1, 1.0)
        assert _lib.load().spx_linear_attention_workspace(dims) > 2 * len(lens) * H * dk * dv * 4
    q, k, v, a, state = _inputs(1, cu[-1], H, kv, dk, dv, n=len(lens), init=True)
    g = torch.Generator(device=DEV).manual_seed(2)
    do = torch.randn(1, cu[-1], H, dv, generator=g, device=DEV).to(torch.bfloat16)
    ds = torch.randn(len(lens), H, dk, dv, generator=g, device=DEV)

    def call(spoilt):
        ins = [t.clone() for t in (q, k, v, a)]
        dout = do.clone()
        if spoilt:
            for i in range(1, len(lens), 2):
                for t in (*ins, dout):
                    t[:, cu[i]:cu[i + 1]] = bad
        ins = [t.requires_grad_(True) for t in (*ins, state.clone())]
        out, last = linear_attention(*ins[:4], initial_state=ins[4], cu_seqlens=cut, return_state=True)
        grads = torch.autograd.grad((out, last), ins, (dout, ds))
        return (out, *grads[:4]), (last, grads[4])

    rows, states = call(False)
    rows2, states2 = call(True)
    assert linear_attention_status() == 0
    here = torch.zeros(cu[-1], dtype=torch.bool, device=DEV)
    for i in range(0, len(lens), 2):
        here[cu[i]:cu[i + 1]] = True
    for x, y in zip(rows, rows2):
        assert torch.isfinite(x[:, here].float()).all() and torch.equal(x[:, here], y[:, here])
    for x, y in zip(states, states2):
        assert torch.isfinite(x[::2]).all() and torch.equal(x[::2], y[::2])
