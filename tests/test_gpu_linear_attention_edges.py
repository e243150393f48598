"""Linear attention at its borders: neighbours in a packed row, rows of no sequence, views, autograd."""

from __future__ import annotations

import math
import subprocess
import sys

import pytest
import torch

from spalmer_b200 import _lib, linear_attention, linear_attention_status, linear_attention_step
from tests.conftest import ROOT
from tests.test_gpu_linear_attention import DEV, _check_forward, _check_gradients, _inputs

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


@pytest.fixture
def dirty(monkeypatch):
    """torch.empty and empty_like hand out memory that somebody else has left NaN in."""

    def spoilt(make):
        def made(*args, **kw):
            t = make(*args, **kw)
            return t.fill_(255 if t.dtype == torch.uint8 else math.nan) if t.is_cuda else t
        return made

    for name in ("empty", "empty_like"):
        monkeypatch.setattr(torch, name, spoilt(getattr(torch, name)))


def _train(q, k, v, a, state, cu, do, ds):
    ins = [t.detach().clone().requires_grad_(True) for t in (q, k, v, a, state)]
    out, last = linear_attention(*ins[:4], initial_state=ins[4], return_state=True,
                                 cu_seqlens=torch.tensor(cu, device=DEV, dtype=torch.int32))
    dq, dk, dv, da, d_state = torch.autograd.grad((out, last), ins, (do, ds), allow_unused=True)
    return (out.detach(), dq, dk, dv, da), (last.detach(), d_state)


@pytest.mark.parametrize("decay", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,kv,dk,dv", [(3, 3, 64, 64), (4, 2, 128, 72)])
@pytest.mark.parametrize("T,cu", [(400, [5, 70, 70, 300]), (300, [10, 200]), (300, [0, 300]), (64, [64, 64]), (40, [7]),
                                  (5003, list(range(1, 5001)))])
def test_tokens_of_no_sequence(dirty, T, cu, H, kv, dk, dv, decay):
    """Rows that a packed call does not cover are zero, gradients too; the others are those of the row cut to them."""

    n = len(cu) - 1
    q, k, v, a, state = _inputs(1, T, H, kv, dk, dv, n=n or 1, init=True, decay=decay)
    state = state[:n]
    g = torch.Generator(device=DEV).manual_seed(3)
    do = torch.randn(1, T, H, dv, generator=g, device=DEV).to(torch.bfloat16)
    ds = torch.randn(n, H, dk, dv, generator=g, device=DEV)
    rows, states = _train(q, k, v, a, state, cu, do, ds)
    assert linear_attention_status() == 0
    lo, hi = cu[0], cu[-1]
    for x in rows:
        assert not x[:, :lo].any() and not x[:, hi:].any()
    if hi > lo:
        cut = [t[:, lo:hi] for t in (q, k, v, a)]
        want_rows, want_states = _train(*cut, state, [c - lo for c in cu], do[:, lo:hi], ds)
        for x, y in zip((*(x[:, lo:hi] for x in rows), *states), (*want_rows, *want_states)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("with_state", [True, False])
@pytest.mark.parametrize("H,kv", [(2, 2), (4, 1)])
def test_unsound_sequences_are_empty_ones(dirty, H, kv, with_state):
    """Sequence 1 runs backwards, sequence 3 past the end: their states pass through, their rows are zero."""

    cu = [0, 100, 50, 200, 400]
    q, k, v, a, state = _inputs(1, 300, H, kv, 64, 64, n=4, init=True)
    cut = torch.tensor(cu, device=DEV, dtype=torch.int32)
    ins = [t.requires_grad_(True) for t in (q, k, v, a)] + ([state.requires_grad_(True)] if with_state else [])
    out, last = linear_attention(*ins[:4], initial_state=state if with_state else None, cu_seqlens=cut, return_state=True)
    g = torch.Generator(device=DEV).manual_seed(3)
    do = torch.randn(out.shape, generator=g, device=DEV).to(torch.bfloat16)
    ds = torch.randn(last.shape, generator=g, device=DEV)
    grads = torch.autograd.grad((out, last), ins, (do, ds))
    assert linear_attention_status() != 0
    for x in (out, *grads[:4]):
        assert torch.isfinite(x.float()).all() and not x[:, 200:].any()
    assert torch.isfinite(last).all()
    for i in (1, 3):
        assert torch.equal(last[i], state[i] if with_state else torch.zeros_like(last[i]))
        if with_state:  # through 1 / scale and scale
            assert torch.allclose(grads[4][i], ds[i], rtol=2.0 ** -22, atol=0)


def test_states_off_sixteen_bytes():
    """An initial state, and a last state's gradient, one element behind a 16-byte boundary."""

    q, k, v, a, state = _inputs(2, 150, 2, 1, 64, 72, init=True)
    g = torch.Generator(device=DEV).manual_seed(8)
    ds = torch.randn(state.shape, generator=g, device=DEV)

    def off(t):
        moved = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:].view(t.shape)
        moved.copy_(t)
        assert moved.data_ptr() % 16
        return moved

    def call(move):
        ins = [t.detach().requires_grad_(True) for t in (q, k, v, a, move(state))]
        out, last = linear_attention(*ins[:4], initial_state=ins[4], return_state=True)
        return out, last, *torch.autograd.grad((out, last), ins, (torch.ones_like(out), move(ds)))

    for got, want in zip(call(off), call(lambda t: t)):
        assert torch.equal(got, want)


FIRST_CALL = """
import torch
from spalmer_b200 import linear_attention, linear_attention_status

q, k, v = (torch.randn(1, 300, 2, 64, device="cuda").to(torch.bfloat16) for _ in range(3))
a = -torch.rand(1, 300, 2, device="cuda")
cu = torch.tensor([0, 100, 50, 300], device="cuda", dtype=torch.int32)  # sequence 1 runs backwards
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out, _ = linear_attention(q, k, v, a, cu_seqlens=cu)
graph.replay()
torch.cuda.synchronize()
cu.copy_(torch.tensor([0, 100, 200, 300]))
graph.replay()
torch.cuda.synchronize()
assert linear_attention_status(clear=False) != 0, "a later replay has cleared the status"
assert linear_attention_status() != 0 and linear_attention_status() == 0
graph.replay()
torch.cuda.synchronize()
assert linear_attention_status() == 0
want, _ = linear_attention(q, k, v, a, cu_seqlens=cu)
assert torch.equal(out, want)
"""


def test_first_call_inside_a_graph():
    """The status word outlives a graph whose capture made the first call, and no replay clears it."""

    done = subprocess.run([sys.executable, "-c", FIRST_CALL], cwd=ROOT, capture_output=True, text=True, timeout=120)
    assert done.returncode == 0, done.stderr


@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 72)])
@pytest.mark.parametrize("at", [0, 1, 31, 40, 70, 127, 128, 250, 299])
def test_a_nan_decay_stays_on_its_side(at, dk, dv):
    """The decay of a token is between it and those before: they keep their outputs and d q, it and those after it
    their d k and d v.  They are those of a token that forgets everything, whose block takes the same sums."""

    q, k, v, a, _ = _inputs(2, 300, 2, 2, dk, dv)
    g = torch.Generator(device=DEV).manual_seed(1)
    do = torch.randn(2, 300, 2, dv, generator=g, device=DEV).to(torch.bfloat16)

    def call(a):
        ins = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = linear_attention(*ins, a)[0]
        return out.detach(), *torch.autograd.grad(out, ins, do)

    spoilt, forgets = a.clone(), a.clone()
    spoilt[:, at], forgets[:, at] = math.nan, -math.inf
    for i, (got, want) in enumerate(zip(call(spoilt), call(forgets))):
        keep = slice(None, at) if i < 2 else slice(at, None)
        assert torch.isfinite(want.float()).all() and torch.equal(got[:, keep], want[:, keep])
        if at:
            assert torch.isnan(got[:, at:] if i < 2 else got[:, :at]).any()


@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 72)])
@pytest.mark.parametrize("resets", [(27,), (0, 5, 9, 30), tuple(range(26)), tuple(range(0, 32, 3))])
@pytest.mark.parametrize("strong", [-math.inf, -150.0, -60.0])
def test_many_strong_decays_in_a_block(strong, resets, dk, dv):
    """Tokens that forget (nearly) everything, up to 26 of a block of 32, with mild ones after and between them."""

    q, k, v, a, state = _inputs(1, 300, 2, 1, dk, dv, init=True, span=(50.0, 300.0))
    for block in (0, 64, 160, 224, 256):
        a[:, [block + r for r in resets]] = strong
    _check_forward(q, k, v, a, state)
    _check_gradients(q, k, v, a, None)  # the first state's gradient has passed all of them: below FP32's range


def _odd_views(q, k, v):
    """The same values as views of one leaf: off 16 bytes, and no stride of tokens or heads a multiple of 16 bytes."""

    lead, width = q.shape[:-2], max(q.shape[-1], v.shape[-1])
    heads = q.shape[-2] + 2 * k.shape[-2]
    wide = torch.zeros(math.prod(lead) * heads * (width + 1) + 3, device=DEV, dtype=torch.bfloat16)
    rows = wide[3:].view(*lead, heads, width + 1)
    at = 0
    for t in (q, k, v):
        rows[..., at:at + t.shape[-2], :t.shape[-1]] = t
        at += t.shape[-2]
    wide.requires_grad_(True)
    rows = wide[3:].view(*lead, heads, width + 1)
    at, views = 0, []
    for t in (q, k, v):
        view = rows[..., at:at + t.shape[-2], :t.shape[-1]]
        assert torch.equal(view, t) and view.data_ptr() % 16 and view.stride(-2) % 8
        views.append(view)
        at += t.shape[-2]
    return wide, views


@pytest.mark.parametrize("B,T,H,kv,dk,dv", [(2, 300, 4, 2, 64, 64), (1, 5, 3, 3, 40, 128), (2, 150, 2, 1, 128, 72)])
def test_misaligned_views(B, T, H, kv, dk, dv):
    q, k, v, a, state = _inputs(B, T, H, kv, dk, dv, init=True)
    g = torch.Generator(device=DEV).manual_seed(1)
    do = torch.randn(B, T, H, dv, generator=g, device=DEV).to(torch.bfloat16)
    ins = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out, last = linear_attention(*ins, a, initial_state=state, return_state=True)
    want = torch.autograd.grad(out, ins, do)
    wide, views = _odd_views(q, k, v)
    odd = torch.empty(do.numel() + 1, dtype=do.dtype, device=DEV)[1:].view(do.shape).copy_(do)
    out2, last2 = linear_attention(*views, a, initial_state=state, return_state=True)
    assert torch.equal(out2, out) and torch.equal(last2, last)
    for x, y in zip(torch.autograd.grad(out2, views, odd, retain_graph=True), want):
        assert torch.equal(x, y)
    (whole,) = torch.autograd.grad(out2, wide, odd)
    assert torch.equal(whole.sort().values, torch.cat([*(y.flatten() for y in want), whole.new_zeros(
        whole.numel() - sum(y.numel() for y in want))]).sort().values)


def test_misaligned_views_of_a_step():
    q, k, v, a, state = _inputs(1, 5, 4, 2, 64, 72, n=5, init=True)
    q, k, v, a = q[0], k[0], v[0], a[0]
    _, views = _odd_views(q, k, v)
    other = state.clone()
    want = linear_attention_step(q, k, v, a, state)
    assert torch.equal(linear_attention_step(*(t.detach() for t in views), a, other), want)
    assert torch.equal(other, state)
