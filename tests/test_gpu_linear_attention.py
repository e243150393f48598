"""Linear attention with a decay per head against the token-by-token recurrence
in 64 bits: batched and packed sequences, carried states, shared heads, strong
decays, segments of long sequences, gradients, and single tokens.

Tolerances (unit: the half ulp of BF16, 2^-8 of a value at most, 2^-8 / sqrt(3)
in the root mean square over many).
* out rounds the decayed q . k, the state and the result once each: the sums of
  products carry at most one unit of the sum of their magnitudes, and in the
  mean, as independent errors, sqrt(2) units of the result.
* gradients multiply operands split into two BF16 parts (2^-16): one unit.
* the last state is a sum of FP32 products and decays: 2^-24 a rounding, some
  dozens of them; an error of 1e-5 of its norm allows for a hundred.
* d log decay is a running sum over the sequence of q . dq - k . dk, whose
  terms carry 2^-14 of the magnitudes of what they sum; independent errors add
  up as the root of the sum of squares (times 4).
Few elements or rounding at unlucky places are allowed for by SLACK."""

from __future__ import annotations

import math

import pytest
import torch

from spalmer_b200 import linear_attention, linear_attention_status, linear_attention_step
from tests.token_reference import HALF_ULP, MEAN_ULP, attention, rel

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
SLACK = 1.15


def _inputs(B, T, H, kv, dk, dv, *, n=None, init=False, decay=torch.float32, span=(4.0, 300.0), seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + 131 * T + 7 * H + dk + dv)

    def rnd(*shape):
        return torch.randn(shape, generator=g, device=DEV).to(torch.bfloat16)

    u = torch.rand(H, generator=g, device=DEV)
    spans = torch.exp(math.log(span[0]) + u * (math.log(span[1]) - math.log(span[0])))
    a = (-torch.exp(0.5 * torch.randn(B, T, H, generator=g, device=DEV)) / spans).to(decay)
    state = 2 * torch.randn(n or B, H, dk, dv, generator=g, device=DEV) if init else None
    return rnd(B, T, H, dk), rnd(B, T, kv, dk), rnd(B, T, kv, dv), a, state


def _check_forward(q, k, v, a, state, cu=None, scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    cut = None if cu is None else torch.tensor(cu, device=DEV, dtype=torch.int32)
    out, last = linear_attention(q, k, v, a, scale=scale, initial_state=state, cu_seqlens=cut, return_state=True)
    assert linear_attention_status() == 0
    wide = [t.detach().double() for t in (q, k, v, a)]
    s64 = None if state is None else state.detach().double()
    want, want_last = attention(*wide, s64, scale, cu)
    size, _ = attention(*(t.abs() for t in wide[:3]), wide[3], None if s64 is None else s64.abs(), abs(scale), cu)
    assert out.shape == want.shape and out.dtype == torch.bfloat16 and last.dtype == torch.float32
    assert torch.all((out.double() - want).abs() <= HALF_ULP * want.abs() + 1.01 * HALF_ULP * size + 1e-30)
    if want.numel() >= 4096:
        assert rel(out, want) <= SLACK * math.sqrt(2) * MEAN_ULP
    if want_last.numel():
        assert rel(last, want_last) <= 1e-5
    return out, last


CASES = {
    # name: (B, T, H, kv, dk, dv, options)
    "one_token": (2, 1, 3, 3, 64, 64, {}),
    "few_tokens": (3, 8, 2, 1, 64, 32, {"init": True}),
    "nine_tokens": (1, 9, 2, 2, 64, 64, {"init": True}),
    "chunk_less_one": (1, 127, 2, 2, 64, 64, {}),
    "chunk": (1, 128, 1, 1, 64, 64, {"init": True}),
    "chunk_and_one": (2, 129, 2, 2, 128, 128, {"init": True}),
    "narrow": (1, 300, 4, 1, 8, 128, {"decay": torch.bfloat16}),
    "narrow_value": (1, 300, 2, 2, 128, 8, {"init": True}),
    "odd_widths": (2, 200, 4, 2, 72, 40, {"init": True}),
    "wide_value": (1, 260, 2, 2, 64, 120, {}),
    "many": (50, 150, 4, 2, 64, 64, {}),
    "long": (1, 5000, 1, 1, 128, 128, {"init": True}),
    "long_two": (2, 3000, 2, 1, 64, 64, {"init": True, "decay": torch.bfloat16}),
    "strong_decay": (1, 700, 2, 2, 64, 64, {"init": True, "span": (0.02, 1.0)}),
    "hardly_any_decay": (1, 1500, 2, 2, 64, 64, {"span": (1e4, 1e6)}),
}


@pytest.mark.parametrize("name", CASES)
def test_forward(name):
    B, T, H, kv, dk, dv, opt = CASES[name]
    _check_forward(*_inputs(B, T, H, kv, dk, dv, **opt))


PACKED = {
    "ends_everywhere": (500, [0, 1, 1, 130, 200, 456, 500]),
    "single": (77, [0, 77]),
    "ones": (40, list(range(41))),
    "empty_ends": (128, [0, 0, 0, 128, 128]),
    "chunks": (512, [0, 128, 384, 512]),
    "long": (4100, [0, 3, 4000, 4100]),
}


@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 72)])
@pytest.mark.parametrize("name", PACKED)
def test_packed(name, dk, dv):
    T, cu = PACKED[name]
    _check_forward(*_inputs(1, T, 3, 3, dk, dv, n=len(cu) - 1, init=True), cu=cu)


def _check_gradients(q, k, v, a, state, cu=None, through="both", scale=None):
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    ins = [t.detach().requires_grad_(True) for t in (q, k, v, a)] + ([state.detach().requires_grad_(True)] if state is not None else [])
    cut = None if cu is None else torch.tensor(cu, device=DEV, dtype=torch.int32)
    out, last = linear_attention(*ins[:4], scale=scale, initial_state=ins[4] if state is not None else None,
                                 cu_seqlens=cut, return_state=True)
    g = torch.Generator(device=DEV).manual_seed(5)
    do = torch.randn(out.shape, generator=g, device=DEV).to(torch.bfloat16)
    ds = torch.randn(last.shape, generator=g, device=DEV)
    outs, grads = {"both": ((out, last), (do, ds)), "out": ((out,), (do,)), "state": ((last,), (ds,))}[through]
    got = torch.autograd.grad(outs, ins, grads, allow_unused=True)
    assert linear_attention_status() == 0
    wide = [t.detach().double().requires_grad_(True) for t in ins]
    o64, s64 = attention(*wide[:4], wide[4] if state is not None else None, scale, cu)
    outs = {"both": (o64, s64), "out": (o64,), "state": (s64,)}[through]
    want = torch.autograd.grad(outs, wide, [x.double() for x in grads], allow_unused=True)
    for name, x, y in zip(("q", "k", "v"), got, want):
        if y is None or not y.any():
            assert x is None or not x.any(), name
            continue
        assert x.dtype == torch.bfloat16 and x.shape == y.shape
        assert rel(x, y) <= SLACK * MEAN_ULP, name
        worst = float((x.double() - y).abs().max() / y.abs().max())
        assert worst <= 2 * HALF_ULP, name
    # d log decay: the terms of the running sum, per query head
    group = q.shape[2] // k.shape[2]
    wide2 = [wide[0], *(t.detach().repeat_interleave(group, 2).requires_grad_(True) for t in wide[1:3]), wide[3]]
    o2, s2 = attention(*wide2, wide[4] if state is not None else None, scale, cu)
    outs = {"both": (o2, s2), "out": (o2,), "state": (s2,)}[through]
    gq, gk = torch.autograd.grad(outs, [wide2[0], wide2[1]], [x.double() for x in grads], allow_unused=True)
    m = wide2[1].detach().abs() * gk.abs()
    if gq is not None:
        m = torch.cat((m, wide2[0].detach().abs() * gq.abs()), -1)
    noise = m.sum(-1).square().sum(1, keepdim=True).sqrt()  # [B, 1, H]: over the whole row, a bound for every token
    if through != "out":
        noise = noise + (s64.detach() * ds.double()).flatten(2).square().sum(-1).sqrt().amax(0)[None, None]
    unit = HALF_ULP if a.dtype == torch.bfloat16 else 0.0
    assert got[3].dtype == a.dtype
    assert torch.all((got[3].double() - want[3]).abs() <= unit * want[3].abs() + 4 * 2.0 ** -14 * noise)
    if state is not None:
        assert rel(got[4], want[4]) <= 4 * 2.0 ** -16
    return got


@pytest.mark.parametrize("through", ["both", "out", "state"])
@pytest.mark.parametrize("name", ["one_token", "few_tokens", "nine_tokens", "chunk_and_one", "narrow", "odd_widths",
                                  "wide_value", "long_two", "strong_decay"])
def test_gradients(name, through):
    B, T, H, kv, dk, dv, opt = CASES[name]
    _check_gradients(*_inputs(B, T, H, kv, dk, dv, **opt), through=through)


@pytest.mark.parametrize("kv", [4, 1])
@pytest.mark.parametrize("name", PACKED)
def test_packed_gradients(name, kv):
    T, cu = PACKED[name]
    _check_gradients(*_inputs(1, T, 4, kv, 64, 128, n=len(cu) - 1, init=True), cu=cu)


# more sequences and heads than SMs, in numbers that whole ones do not fill: the kernel cuts some in two
@pytest.mark.parametrize("B,T,H,kv,dk,dv", [(13, 300, 12, 6, 64, 64), (5, 700, 8, 8, 128, 128), (75, 129, 2, 2, 64, 32),
                                            (41, 517, 4, 1, 40, 104)])
def test_even_shares(B, T, H, kv, dk, dv):
    q, k, v, a, state = _inputs(B, T, H, kv, dk, dv, init=True)
    first = _check_forward(q, k, v, a, state)
    again = _check_forward(q, k, v, a, state)
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    _check_gradients(q, k, v, a, state)


# every CTA takes many short and empty sequences one after another
@pytest.mark.parametrize("dk,dv", [(64, 64), (128, 72)])
@pytest.mark.parametrize("lengths", [(0, 0, 0, 1, 2, 5, 40, 129, 300), (0, 0, 0, 0, 0, 0, 0, 1), (0, 3), (1, 2)])
def test_packed_short_and_empty(lengths, dk, dv):
    g = torch.Generator().manual_seed(dk + len(lengths))
    lens = [lengths[i] for i in torch.randint(len(lengths), (300,), generator=g).tolist()]
    cu = [0] + torch.tensor(lens).cumsum(0).tolist()
    q, k, v, a, state = _inputs(1, cu[-1], 4, 2, dk, dv, n=len(lens), init=True)
    for _ in range(3):
        _check_forward(q, k, v, a, state, cu=cu)
    _check_gradients(q, k, v, a, state, cu=cu)


@pytest.mark.parametrize("cu", [[0, 9000, 9000, 9000, 9000, 9003, 9003], [0, 0, 0, 0, 0, 7000]])
def test_packed_long_among_empty(cu):
    q, k, v, a, state = _inputs(1, cu[-1], 2, 2, 64, 64, n=len(cu) - 1, init=True)
    _check_forward(q, k, v, a, state, cu=cu)


@pytest.mark.parametrize("T,cu", [(1, None), (5, None), (130, None), (9, [0, 1, 2, 6, 6, 9])])
def test_first_token_has_no_decay_gradient(T, cu):
    q, k, v, a, _ = _inputs(3 if cu is None else 1, T, 4, 2, 96, 128)
    a = a.requires_grad_(True)
    cut = None if cu is None else torch.tensor(cu, device=DEV, dtype=torch.int32)
    out, last = linear_attention(q, k, v, a, cu_seqlens=cut, return_state=True)
    (da,) = torch.autograd.grad([out, last], a, [torch.randn_like(out), torch.randn_like(last)])
    first = [0] if cu is None else cu[:-1]
    assert torch.all(da[:, first] == 0.0)


def test_gradients_against_differences():
    """The last state is linear in k and v and smooth in the decays, and comes back in
    FP32; the output is linear in q: central differences of the operator itself."""

    q, k, v, a, s = _inputs(1, 200, 2, 1, 64, 64, init=True, seed=3)
    g = torch.Generator(device=DEV).manual_seed(9)
    c = torch.randn(1, 2, 64, 64, generator=g, device=DEV)
    ins = [t.requires_grad_(True) for t in (k, v, a, s)]
    last = linear_attention(q, ins[0], ins[1], ins[2], initial_state=ins[3], return_state=True)[1]
    grads = torch.autograd.grad(last, ins, c)

    def value(args):
        with torch.no_grad():
            return float((linear_attention(q, *args[:3], initial_state=args[3], return_state=True)[1].double() * c).sum())

    base = [t.detach() for t in (k, v, a, s)]
    for i, (t, grad) in enumerate(zip(base, grads)):
        if i == 2:
            d, step = torch.randn(t.shape, generator=g, device=DEV), 1e-2
            near = [t - step * d * t, t + step * d * t]  # decays stay negative
            d = d * t
        else:  # a direction that BF16 inputs take exactly: some elements are doubled, or vanish
            pick = (torch.rand(t.shape, generator=g, device=DEV) < 0.1).to(t.dtype)
            d, step = t * pick, 1.0
            near = [t - d, t + d]
        ends = [value([*base[:i], x, *base[i + 1:]]) for x in near]
        want = (ends[1] - ends[0]) / (2 * step)
        dot = float((grad.double() * d.double()).sum())
        size = float((grad.double().abs() * d.double().abs()).sum())
        noise = 2e-5 * float(last.detach().double().norm() * c.double().norm()) / step  # the two values' own error
        curve = 2e-3 * size if i == 2 else 0.0  # the second-order term of exp over steps of a hundredth
        assert abs(dot - want) <= HALF_ULP * size + noise + curve
    # q, through the output
    qg = q.detach().requires_grad_(True)
    out = linear_attention(qg, *base[:3], initial_state=base[3])[0]
    do = torch.randn(out.shape, generator=g, device=DEV).to(torch.bfloat16)
    dq, = torch.autograd.grad(out, qg, do)
    zero = linear_attention(torch.zeros_like(q), *base[:3], initial_state=base[3])[0]
    assert not zero.any()
    want = float((out.detach().double() * do.double()).sum())  # linear: the value is the derivative along q
    slack = 3 * HALF_ULP * float((out.detach().double().square() * do.double().square()).sum().sqrt())
    slack += HALF_ULP * float((dq.double() * q.detach().double()).square().sum().sqrt()) * 3
    assert abs(float((dq.double() * q.detach().double()).sum()) - want) <= slack


def test_resets_and_non_finite_neighbours():
    """A log decay of -inf forgets everything before; NaN and infinity in one packed
    sequence reach no other, wherever the sequences end inside a chunk."""

    q, k, v, a, _ = _inputs(1, 400, 2, 2, 64, 64)
    cu = [0, 70, 71, 150, 333, 400]
    for start in cu[1:-1]:
        a[:, start] = -math.inf
    whole, last = linear_attention(q, k, v, a, return_state=True)
    a2 = a.clone()
    parts, lasts = linear_attention(q, k, v, a2, cu_seqlens=torch.tensor(cu, device=DEV, dtype=torch.int32), return_state=True)
    want, want_last = attention(*(t.double() for t in (q, k, v, a)), None, 64 ** -0.5, cu)
    for got in (whole, parts):
        assert rel(got, want) <= SLACK * math.sqrt(2) * MEAN_ULP
    assert rel(last, want_last[-1:]) <= 1e-5 and rel(lasts, want_last) <= 1e-5
    for bad in (math.nan, math.inf, -math.inf):
        for t in (q, k, v):
            x = t.clone()
            x[:, cu[2]:cu[3]] = bad
            args = [x if u is t else u for u in (q, k, v)]
            o, s = linear_attention(*args, a, cu_seqlens=torch.tensor(cu, device=DEV, dtype=torch.int32), return_state=True)
            for i in (0, 1, 3, 4):
                assert torch.equal(o[:, cu[i]:cu[i + 1]], parts[:, cu[i]:cu[i + 1]])
                assert torch.equal(s[i], lasts[i])
    assert linear_attention_status() == 0


def test_views_streams_and_repetition():
    """Views of a fused projection equal their copies; a call on another stream and a second call give the same bits."""

    g = torch.Generator(device=DEV).manual_seed(1)
    qkv = torch.randn(2, 333, 8 * 64, generator=g, device=DEV).to(torch.bfloat16)
    q, k, v = qkv[..., :256].unflatten(-1, (4, 64)), qkv[..., 256:384].unflatten(-1, (2, 64)), qkv[..., 384:].unflatten(-1, (2, 64))
    a = -torch.rand(2, 4, 333, generator=g, device=DEV).transpose(1, 2)
    first = linear_attention(q, k, v, a, return_state=True)
    copies = linear_attention(q.contiguous(), k.contiguous(), v.contiguous(), a.contiguous(), return_state=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = linear_attention(q, k, v, a, return_state=True)
    side.synchronize()
    moved = linear_attention(*(qkv.roll(1, -1)[..., 1:].clone() if t is None else t for t in (q, k, v)), a, return_state=True)
    expanded = linear_attention(q[:1].expand(2, -1, -1, -1), k[:1].expand(2, -1, -1, -1), v[:1].expand(2, -1, -1, -1),
                                a[:1].expand(2, -1, -1), return_state=True)
    for pair in zip(first, copies):
        assert torch.equal(*pair)
    for pair in zip(first, other):
        assert torch.equal(*pair)
    for pair in zip(first, moved):
        assert torch.equal(*pair)
    assert torch.equal(expanded[0][0], first[0][0]) and torch.equal(expanded[0][1], first[0][0])
    ins = [t.detach().requires_grad_(True) for t in (q, k, v, a)]
    out = linear_attention(*ins)[0]
    do = torch.randn(out.shape, generator=g, device=DEV).to(torch.bfloat16)
    one, two = (torch.autograd.grad(linear_attention(*ins)[0], ins, do) for _ in range(2))
    for pair in zip(one, two):
        assert torch.equal(*pair)


def test_graph_capture():
    """The chunked forward in a CUDA graph: nothing is allocated or synchronised by the library."""

    q, k, v, a, s = _inputs(1, 3000, 2, 2, 64, 64, init=True)
    want = linear_attention(q, k, v, a, initial_state=s, return_state=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = linear_attention(q, k, v, a, initial_state=s, return_state=True)
    graph.replay()
    torch.cuda.synchronize()
    for pair in zip(got, want):
        assert torch.equal(*pair)


def test_empty_sequences():
    q, k, v, a, s = _inputs(3, 0, 2, 2, 64, 64, init=True)
    out, last = linear_attention(q, k, v, a, initial_state=s, return_state=True)
    assert out.shape == (3, 0, 2, 64) and torch.equal(last, s)
    out, last = linear_attention(q[:0], k[:0], v[:0], a[:0], return_state=True)
    assert out.shape == (0, 0, 2, 64) and last.shape == (0, 2, 64, 64)
    out, last = linear_attention(q[:1], k[:1], v[:1], a[:1], cu_seqlens=torch.zeros(3, device=DEV, dtype=torch.int32),
                                 initial_state=s[:2], return_state=True)
    assert torch.equal(last, s[:2])
    assert linear_attention_status() == 0


def test_unsound_offsets_are_recorded():
    """Offsets out of order or out of range: their sequences are skipped, the others are right, the status says so."""

    q, k, v, a, _ = _inputs(1, 300, 2, 2, 64, 64)
    cu = [0, 100, 50, 200, 400]  # sequence 1 runs backwards, sequence 3 past the end
    out, _ = linear_attention(q, k, v, a, cu_seqlens=torch.tensor(cu, device=DEV, dtype=torch.int32), return_state=True)
    assert linear_attention_status() != 0
    assert linear_attention_status() == 0  # cleared
    # sequence 2 (tokens 50 .. 200) overlaps sequence 0; its own tail belongs to it alone
    want, _ = attention(*(t.double() for t in (q[:, 50:200], k[:, 50:200], v[:, 50:200], a[:, 50:200])), None, 64 ** -0.5)
    assert rel(out[:, 100:200], want[:, 50:]) <= SLACK * math.sqrt(2) * MEAN_ULP


# ---------------------------------------------------------------- single tokens
@pytest.mark.parametrize("slots", [None, "some"])
@pytest.mark.parametrize("B,H,kv,dk,dv", [(1, 1, 1, 8, 8), (1, 12, 12, 64, 64), (5, 4, 2, 72, 40), (3, 8, 1, 128, 120),
                                          (33, 4, 4, 128, 128), (2, 2, 2, 16, 128), (2, 2, 2, 128, 16)])
def test_step(B, H, kv, dk, dv, slots):
    """FP32 arithmetic: 2^-24 a rounding, at most dk of them a sum; the output rounds once."""

    q, k, v, a, _ = _inputs(1, B, H, kv, dk, dv, decay=torch.float32 if slots else torch.bfloat16)
    q, k, v, a = q[0], k[0], v[0], a[0]
    g = torch.Generator(device=DEV).manual_seed(1)
    n = B + 3
    state = torch.randn(n, H, dk, dv, generator=g, device=DEV)
    at = torch.randperm(n, generator=torch.Generator().manual_seed(B))[:B].to(DEV) if slots else None
    if slots and B >= 3:
        at[1], at[2] = -1, n + 5
    before = state.clone()
    out = linear_attention_step(q, k, v, a, state, slots=at)
    rows = torch.arange(B, device=DEV) if at is None else at
    live = (rows >= 0) & (rows < n)
    idx = rows[live]
    group = H // kv
    want = before[idx].double() * torch.exp(a[live].double())[..., None, None] + (
        k[live].double().repeat_interleave(group, 1)[..., None] * v[live].double().repeat_interleave(group, 1)[:, :, None])
    o = dk ** -0.5 * (q[live].double()[:, :, None] @ want)[:, :, 0]
    size = dk ** -0.5 * (q[live].double().abs()[:, :, None] @ want.abs())[:, :, 0]
    assert torch.all((state[idx].double() - want).abs() <= 2.0 ** -22 * (want.abs() + before[idx].double().abs()))
    assert torch.all((out[live].double() - o).abs() <= HALF_ULP * o.abs() + 2.0 ** -16 * size)
    assert not out[~live].any()
    rest = torch.ones(n, dtype=torch.bool, device=DEV)
    rest[idx] = False
    assert torch.equal(state[rest], before[rest])


def test_step_continues_a_prompt():
    """A prompt's last state, then token by token, equals the whole sequence at once."""

    q, k, v, a, _ = _inputs(2, 140, 4, 2, 64, 64)
    out, state = linear_attention(q[:, :133], k[:, :133], v[:, :133], a[:, :133], return_state=True)
    want, want_last = attention(*(t.double() for t in (q, k, v, a)), None, 64 ** -0.5)
    for t in range(133, 140):
        o = linear_attention_step(q[:, t], k[:, t], v[:, t], a[:, t], state)
        assert rel(o, want[:, t]) <= 2 * MEAN_ULP
    assert rel(state, want_last) <= 1e-5


def test_step_far_slots():
    """A state whose element offset passes 2^31."""

    H, d = 16, 128
    slots = 2 ** 31 // (H * d * d) + 2
    state = torch.zeros(slots, H, d, d, device=DEV)
    q, k, v, a, _ = _inputs(1, 2, H, H, d, d)
    at = torch.tensor([slots - 1, 0], device=DEV)
    out = linear_attention_step(q[0], k[0], v[0], a[0], state, slots=at)
    want = k[0].double()[..., None] * v[0].double()[:, :, None]
    assert torch.allclose(state[at].double(), want, rtol=2.0 ** -22, atol=0)
    o = d ** -0.5 * (q[0].double()[:, :, None] @ want)[:, :, 0]
    assert rel(out, o) <= 1.1 * MEAN_ULP


def test_refusals():
    q, k, v, a, s = _inputs(1, 20, 4, 2, 64, 64, init=True)
    with pytest.raises(ValueError, match="bfloat16"):
        linear_attention(q.float(), k, v, a)
    with pytest.raises(ValueError, match="log_decay"):
        linear_attention(q, k, v, a.double())
    with pytest.raises(ValueError, match="leading"):
        linear_attention(q, k[:, :10], v, a)
    with pytest.raises(ValueError, match="leading"):
        linear_attention(q, k, v, a[..., :2])
    with pytest.raises(ValueError, match="head dimension"):
        linear_attention(q, k[..., :32], v, a)
    with pytest.raises(ValueError, match="multiple"):
        linear_attention(q[:, :, :3], k, v, a[..., :3])
    with pytest.raises(ValueError, match="multiples of 8"):
        linear_attention(q[..., :60], k[..., :60], v, a)
    with pytest.raises(ValueError, match="multiples of 8"):
        wide = torch.zeros(1, 20, 4, 136, device=DEV, dtype=torch.bfloat16)
        linear_attention(wide, wide, wide, a)
    with pytest.raises(ValueError, match="scale"):
        linear_attention(q, k, v, a, scale=0.0)
    with pytest.raises(ValueError, match="initial_state"):
        linear_attention(q, k, v, a, initial_state=s[:, :2])
    with pytest.raises(ValueError, match="cu_seqlens"):
        linear_attention(q, k, v, a, cu_seqlens=torch.tensor([0, 20], device=DEV))
    with pytest.raises(ValueError, match="packed row"):
        two = [t.repeat(2, *[1] * (t.ndim - 1)) for t in (q, k, v, a)]
        linear_attention(*two, cu_seqlens=torch.tensor([0, 20], device=DEV, dtype=torch.int32))
    step = [t[:, 0] for t in (q, k, v, a)]
    with pytest.raises(ValueError, match="state"):
        linear_attention_step(*step, s.transpose(2, 3))
    with pytest.raises(ValueError, match="fewer slots"):
        linear_attention_step(*step, s[:0])
    with pytest.raises(ValueError, match="slots"):
        linear_attention_step(*step, s, slots=torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(NotImplementedError):
        linear_attention_step(step[0].clone().requires_grad_(True), *step[1:], s)
