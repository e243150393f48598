"""Timed cases of the token half of a block: the operators that stand between two channel mixers.

Residual addition with RMSNorm (BF16 or MXFP8 rows out, and its backward pass), rotary positions on queries and
keys, and linear attention with one decay per head: the chunked form for prompts and training, the recurrent form
for single tokens.  ``run`` computes a case in plain 32-bit torch operations, or through the framework where
``own`` is true; ``exact`` restates each operator in 64 bits, token by token.
"""

from __future__ import annotations

import math

import torch
import torch.nn.functional as F

own = False

EPS = 1e-6
CHUNK = 128  # of the plain chunked form


def listed():
    return [
        # residual + norm before the channel mixer of a handful of decoding requests: latency
        dict(name="norm_decode", op="norm", rows=5, d=768, res32=False),
        # the same in a training step of the 100M-preset layer: forward and backward of 65,536 tokens
        dict(name="norm_train", op="norm_train", rows=65536, d=768, res32=False),
        # serving a wider model from 8-bit projections: FP32 residual stream, a ragged number of rows
        dict(name="norm_mxfp8", op="norm_mxfp8", rows=16387, d=2048, res32=True),
        # rotary positions of one decoding step, every request at a position of its own
        dict(name="rope_decode", op="rope", tokens=48, heads=12, kv_heads=12, d=64, rot=64, interleaved=False,
             reach=8192, stretch=1.0),
        # rotary positions of a training step at the 100M-preset width
        dict(name="rope_train", op="rope_train", tokens=65536, heads=12, kv_heads=12, d=64, rot=64, interleaved=False,
             reach=4096, stretch=1.0),
        # a long prompt far beyond the trained context: half of each head rotates, adjacent pairs, few key heads
        dict(name="rope_long", op="rope", tokens=30011, heads=16, kv_heads=4, d=128, rot=64, interleaved=True,
             reach=1000000, stretch=16.0),
        # one request decoding alone
        dict(name="step_one", op="step", batch=1, slots=1, heads=12, kv_heads=12, dk=64, dv=64),
        # a full decoding batch over a cache of states, key heads shared by four query heads
        dict(name="step_batch", op="step", batch=190, slots=256, heads=16, kv_heads=4, dk=128, dv=128),
        # prompts of a serving step, packed: from an empty one and one token to thousands
        dict(name="attn_ragged", op="attn", batch=37, total=20011, packed=True, heads=12, kv_heads=12, dk=64, dv=64,
             carried=True),
        # one very long prompt on few heads: the sequence itself has to be spread over the GPU
        dict(name="attn_prompt", op="attn", batch=1, total=65536, packed=False, heads=6, kv_heads=6, dk=128, dv=128,
             carried=False),
        # a training step of the token mixer at the 100M-preset width
        dict(name="attn_train", op="attn_train", batch=16, total=65536, packed=False, heads=12, kv_heads=12, dk=64,
             dv=64, carried=False),
        # training with wide shared key heads on an odd sequence length
        dict(name="attn_train_shared", op="attn_train", batch=2, total=2 * 4095, packed=False, heads=16, kv_heads=4,
             dk=128, dv=128, carried=False),
    ]


def _log(rng, low, high, multiple=1):
    v = math.exp(rng.uniform(math.log(low), math.log(high + 0.999)))
    v = max(low, min(high, int(v)))
    v = max(multiple, v // multiple * multiple)
    return v + multiple if v == 3072 else v


def draw(rng):
    op = rng.choice(["norm", "norm_train", "norm_mxfp8", "rope", "rope_train", "step", "attn", "attn", "attn_train",
                     "attn_train"])
    if op.startswith("norm"):
        d = _log(rng, 64, 8192, 32 if op == "norm_mxfp8" else 8)
        rows = _log(rng, 1, min(65536, (1 << 25) // d))
        return dict(op=op, rows=rows, d=d, res32=rng.random() < 0.5)
    if op.startswith("rope"):
        kv = rng.choice([1, 2, 3, 4, 8])
        heads = kv * rng.choice([1, 2, 3, 4])
        d = rng.choice([16, 32, 40, 64, 80, 96, 128, 192, 256])
        rot = rng.choice([d, d // 2 // 2 * 2, d // 4 // 2 * 2])
        tokens = _log(rng, 1, min(65536, (1 << 26) // (d * (heads + kv))))
        return dict(op=op, tokens=tokens, heads=heads, kv_heads=kv, d=d, rot=rot, interleaved=rng.random() < 0.5,
                    reach=_log(rng, 16, 1 << 20), stretch=rng.choice([1.0, 1.0, 4.0, 32.0]))
    kv = rng.choice([1, 2, 3, 4, 6])
    heads = kv * rng.choice([1, 1, 2, 4])
    dk = rng.choice([16, 32, 64, 64, 72, 96, 128, 128])
    dv = rng.choice([dk, dk, 32, 64, 120, 128])
    if op == "step":
        batch = _log(rng, 1, min(512, (1 << 25) // (heads * dk * dv)))
        return dict(op=op, batch=batch, slots=batch + rng.randrange(0, 1 + batch // 2), heads=heads, kv_heads=kv,
                    dk=dk, dv=dv)
    most = min(65536, 26_000_000 // (heads * max(dk, dv)))
    packed = rng.random() < 0.4
    batch = _log(rng, 1, 64)
    if packed:
        total = _log(rng, max(batch, 16), most)
    else:
        total = batch * _log(rng, 1, max(1, most // batch))
    return dict(op=op, batch=batch, total=total, packed=packed, heads=heads, kv_heads=kv, dk=dk, dv=dv,
                carried=rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs
def _lengths(total, count, gen):
    """`count` lengths that sum to `total`, spread over their logarithm; of four or more one is empty and one has one token."""
    if count == 1:
        return [total]
    w = torch.exp(torch.rand(count, generator=gen, dtype=torch.float64) * 5.0)
    fixed = {}
    if count >= 4 and total >= count:
        fixed = {count // 2: 0, count // 3: 1}
        for i in fixed:
            w[i] = 0.0
    left = total - sum(fixed.values())
    n = torch.floor(w / w.sum() * left).to(torch.int64)
    for i, v in fixed.items():
        n[i] = v
    n[-1] += total - int(n.sum())
    return n.tolist()


def _decay(gen, device, shape, dtype):
    """Log decays: each head forgets over a span of its own (from a few tokens to a thousand), each token by its input."""
    heads = shape[-1]
    span = torch.exp(torch.rand(heads, generator=gen, device=device) * (math.log(1000.0) - math.log(4.0)) + math.log(4.0))
    g = -torch.exp(0.5 * torch.randn(shape, generator=gen, device=device)) / span
    return g.to(dtype)


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    op = case["op"]

    def rnd(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(shape, generator=gen, device=device) * scale).to(dtype)

    s = {"case": case, "op": op}
    if op.startswith("norm"):
        rows, d = case["rows"], case["d"]
        res_type = torch.float32 if case["res32"] else torch.bfloat16
        s["x"] = rnd(rows, d)
        s["res"] = rnd(rows, d, scale=4.0, dtype=res_type)
        s["w"] = (1.0 + 0.1 * torch.randn(d, generator=gen, device=device)).to(torch.bfloat16)
        if op == "norm_train":
            s["dy"] = rnd(rows, d)
            s["dsum"] = rnd(rows, d, dtype=res_type)
            for name in ("x", "res", "w"):
                s[name].requires_grad_(True)
        return s
    if op.startswith("rope"):
        n, h, kv, d, rot = case["tokens"], case["heads"], case["kv_heads"], case["d"], case["rot"]
        # queries and keys as a fused projection leaves them: two strided views of one tensor
        qkv = rnd(n, h + 2 * kv, d)
        s["q"], s["k"] = qkv[:, :h], qkv[:, h:h + kv]
        s["pos"] = torch.randint(0, case["reach"], (n,), generator=gen, device=device)
        inv = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / max(rot, 1)) / case["stretch"]
        s["freq"] = inv.to(device)
        s["factor"] = 1.0 if case["stretch"] == 1.0 else 0.1 * math.log(case["stretch"]) + 1.0
        if op == "rope_train":
            s["q"], s["k"] = s["q"].detach(), s["k"].detach()
            s["q"].requires_grad_(True)
            s["k"].requires_grad_(True)
            s["dq"], s["dk"] = rnd(n, h, d), rnd(n, kv, d)
        return s
    h, kv, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
    s["scale"] = dk ** -0.5
    if op == "step":
        b, slots = case["batch"], case["slots"]
        s["q"], s["k"], s["v"] = rnd(b, h, dk), rnd(b, kv, dk), rnd(b, kv, dv)
        s["g"] = _decay(gen, device, (b, h), torch.float32)
        s["state"] = rnd(slots, h, dk, dv, scale=3.0, dtype=torch.float32)
        at = torch.randperm(slots, generator=host)[:b]
        if b >= 8:
            at[b // 3] = -1  # a request that has ended: its row of the batch is empty
        s["slots"] = at.to(device)
        return s
    n = case["batch"]
    train = op == "attn_train"
    if case["packed"]:
        lens = _lengths(case["total"], n, host)
        lead = (1, case["total"])
        at = torch.tensor([0] + lens).cumsum(0)
        s["cu"] = at.to(torch.int32).to(device)
        s["longest"] = max(lens)
    else:
        lead = (n, case["total"] // n)
        s["cu"], s["longest"] = None, lead[1]
    s["q"], s["k"], s["v"] = rnd(*lead, h, dk), rnd(*lead, kv, dk), rnd(*lead, kv, dv)
    # training takes its decays from a BF16 projection, serving keeps them in FP32
    s["g"] = _decay(gen, device, (*lead, h), torch.bfloat16 if train else torch.float32)
    s["state"] = rnd(n, h, dk, dv, scale=2.0, dtype=torch.float32) if case["carried"] else None
    if train:
        s["do"] = rnd(*lead, h, dv)
        for name in ("q", "k", "v", "g"):
            s[name].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_norm(x, res, w):
    summed = (x.float() + res.float()).to(res.dtype)
    h = summed.float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * w.float()
    return y, summed


def _plain_norm_backward(summed, w, dy, dsum):
    h, dy = summed.float(), dy.float()
    r = torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS)
    z = dy * w.float()
    dh = r * (z - h * (r * r * (z * h).mean(-1, keepdim=True))) + dsum.float()
    return dh.to(torch.bfloat16), dh.to(summed.dtype), (dy * h * r).sum(0).to(w.dtype)


def _plain_mxfp8(y):
    """E4M3 values and E8M0 scales of blocks of 32: scale 2^ceil(log2(amax / 448))."""
    b = y.reshape(y.shape[0], -1, 32)
    mant, ex = torch.frexp(b.abs().amax(-1) / 448.0)  # amax / 448 = mant * 2^ex, mant in [0.5, 1)
    e = torch.where(mant == 0.5, ex - 1, ex).clamp(-127, 127)
    e = torch.where(mant == 0, torch.full_like(e, -127), e)
    up = torch.where(e == -127, torch.zeros_like(e), -e)
    v = torch.ldexp(b, up[..., None]).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return v.reshape(y.shape), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _plain_rope(x, pos, freq, factor, interleaved):
    rot = 2 * freq.shape[0]
    angle = pos.double()[:, None] * freq  # a position times a frequency needs more than 24 bits
    c, n = (factor * angle.cos()).float()[:, None], (factor * angle.sin()).float()[:, None]
    y = x.float()
    a, b = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
    u, w = a * c - b * n, b * c + a * n
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, y[..., rot:]), -1).to(x.dtype)


def _sums(g):
    """[..., i, j] = g_{j+1} + ... + g_i for i >= j (0 elsewhere)."""
    n = g.shape[-1]
    below = torch.ones(n, n, dtype=torch.bool, device=g.device).tril(-1)
    return torch.where(below, g[..., :, None].expand(*g.shape, n), 0.0).cumsum(-2)


def _plain_attention(q, k, v, g, state, scale):
    """The chunked form, all chunks at once, in 32 bits: [B, T, H, D] in, [B, T, H, Dv] and the last state out."""
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    group = H // k.shape[2]
    C = min(CHUNK, max(1, T))
    N = -(-T // C)
    pad = N * C - T

    def chunks(x):
        return F.pad(x.float(), (0, 0, 0, 0, 0, pad)).reshape(B, N, C, H, -1).permute(0, 3, 1, 2, 4)

    q, k, v = chunks(q), *(chunks(x.float().repeat_interleave(group, 2)) for x in (k, v))
    g = chunks(g[..., None])[..., 0]  # [B, H, N, C]
    inside = torch.exp(_sums(g)).tril()
    out = ((q @ k.transpose(-1, -2)) * inside) @ v
    cum = g.cumsum(-1)
    total = cum[..., -1]
    local = (k * inside[..., -1, :, None]).transpose(-1, -2) @ v
    first = torch.zeros(B, H, 1, dk, dv, device=q.device) if state is None else state[:, :, None]
    local = torch.cat((first, local), 2)
    across = torch.exp(_sums(F.pad(total, (1, 0)))).tril()
    states = (across @ local.flatten(-2)).unflatten(-1, (dk, dv))
    out = out + (q * torch.exp(cum)[..., None]) @ states[:, :, :-1]
    out = (scale * out).permute(0, 2, 3, 1, 4).reshape(B, N * C, H, dv)[:, :T]
    return out, states[:, :, -1]


def _plain_packed(q, k, v, g, state, scale, cu, longest):
    """The same for packed sequences: padded to the longest, computed, and taken apart again."""
    n, total = cu.shape[0] - 1, q.shape[1]
    lens = (cu[1:] - cu[:-1]).long()
    here = torch.arange(longest, device=q.device)
    inside = here < lens[:, None]
    source = (cu[:-1].long()[:, None] + here).clamp(max=total - 1)

    def padded(x):
        y = x[0][source]
        return y * inside.reshape(n, longest, *([1] * (y.ndim - 2))).to(y.dtype)

    out, last = _plain_attention(padded(q), padded(k), padded(v), padded(g), state, scale)
    token = torch.arange(total, device=q.device)
    row = torch.searchsorted(cu.long(), token, right=True) - 1
    return out[row, token - cu.long()[row]][None], last


def _plain_step(s):
    group = s["q"].shape[1] // s["k"].shape[1]
    k, v = s["k"].float().repeat_interleave(group, 1), s["v"].float().repeat_interleave(group, 1)
    there = s["slots"] >= 0
    new = torch.exp(s["g"].float())[..., None, None] * s["state"][s["slots"].clamp(min=0)] + k[..., None] * v[:, :, None]
    out = s["scale"] * (s["q"].float()[:, :, None] @ new)[:, :, 0]
    out = torch.where(there[:, None, None], out, 0.0).to(s["q"].dtype)
    slots = s["state"].shape[0]
    owner = torch.full((slots + 1,), -1, dtype=torch.int64, device=out.device)
    owner.scatter_(0, torch.where(there, s["slots"], slots), torch.arange(out.shape[0], device=out.device))
    owner = owner[:-1]
    s["state"].copy_(torch.where((owner >= 0)[:, None, None, None], new[owner.clamp(min=0)], s["state"]))
    return {"out": out, "state": s["state"]}


# ------------------------------------------------------------------------------------------------ one pass
def run(s):
    op = s["op"]
    if op == "norm" or op == "norm_train":
        if own:
            from spalmer_b200 import add_rms_norm

            y, summed = add_rms_norm(s["x"], s["res"], s["w"], EPS)
        else:
            y, summed = _plain_norm(s["x"].detach(), s["res"].detach(), s["w"].detach())
            y = y.to(torch.bfloat16)
        if op == "norm":
            return {"y": y, "sum": summed}
        if own:
            dx, dres, dw = torch.autograd.grad((y, summed), (s["x"], s["res"], s["w"]), (s["dy"], s["dsum"]))
        else:
            dx, dres, dw = _plain_norm_backward(summed, s["w"].detach(), s["dy"], s["dsum"])
        return {"y": y.detach(), "sum": summed.detach(), "dx": dx, "dres": dres, "dw": dw}
    if op == "norm_mxfp8":
        if own:
            from spalmer_b200 import add_rms_norm_mxfp8

            values, scales, summed = add_rms_norm_mxfp8(s["x"], s["res"], s["w"], EPS)
            values, scales = values.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)
        else:
            y, summed = _plain_norm(s["x"], s["res"], s["w"])
            values, scales = _plain_mxfp8(y)
        return {"values": values, "scales": scales, "sum": summed}
    if op.startswith("rope"):
        if own:
            from spalmer_b200 import rotary_embed

            q, k = rotary_embed(s["q"], s["k"], s["pos"], s["freq"], interleaved=s["case"]["interleaved"],
                                factor=s["factor"])
        else:
            q, k = (_plain_rope(x, s["pos"], s["freq"], s["factor"], s["case"]["interleaved"])
                    for x in (s["q"], s["k"]))
        if op == "rope":
            return {"q": q, "k": k}
        dq, dk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk}
    if op == "step":
        if own:
            from spalmer_b200 import linear_attention_step

            out = linear_attention_step(s["q"], s["k"], s["v"], s["g"], s["state"], slots=s["slots"], scale=s["scale"])
            return {"out": out, "state": s["state"]}
        return _plain_step(s)
    if own:
        from spalmer_b200 import linear_attention

        out, last = linear_attention(s["q"], s["k"], s["v"], s["g"], scale=s["scale"], initial_state=s["state"],
                                     cu_seqlens=s["cu"], return_state=op == "attn")
    else:
        args = (s["q"], s["k"], s["v"], s["g"], s["state"], s["scale"])
        out, last = _plain_attention(*args) if s["cu"] is None else _plain_packed(*args, s["cu"], s["longest"])
        out = out.to(torch.bfloat16)
    if op == "attn":
        return {"out": out, "state": last}
    dq, dk, dv, dg = torch.autograd.grad(out, (s["q"], s["k"], s["v"], s["g"]), s["do"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv, "dg": dg}


def work(case):
    op = case["op"]
    if op.startswith("norm"):
        n, d, r = case["rows"], case["d"], 4 if case["res32"] else 2
        if op == "norm":
            return {"bytes": n * d * (2 + r + r + 2) + 2 * d, "flops": 6 * n * d}
        if op == "norm_mxfp8":
            return {"bytes": n * d * (2 + r + r + 1) + n * d // 32 + 2 * d, "flops": 8 * n * d}
        # in: x, the residual, both gradients; out: the norm, the sum, the inputs' gradient (one tensor if the types agree)
        return {"bytes": n * d * (2 + r + 2 + r + 2 + r + 2 + (r if r == 4 else 0)) + 4 * d, "flops": 18 * n * d}
    if op.startswith("rope"):
        one = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["d"]
        passes = 2 if op == "rope_train" else 1
        return {"bytes": passes * one * 4 + case["tokens"] * 8, "flops": passes * one * 3}
    h, kv, dk, dv = case["heads"], case["kv_heads"], case["dk"], case["dv"]
    if op == "step":
        n = case["batch"]
        return {"bytes": n * (h * dk * dv * 8 + 2 * (h * dk + kv * dk + kv * dv + h * dv) + 4 * h + 8),
                "flops": n * h * dk * dv * 5}
    n = case["total"]
    state = case["batch"] * h * dk * dv * 4
    qkv, o = h * dk + kv * dk + kv * dv, h * dv
    if op == "attn":
        return {"bytes": n * (2 * (qkv + o) + 4 * h) + state * (2 if case["carried"] else 1), "flops": 4 * n * h * dk * dv}
    return {"bytes": n * 2 * (2 * qkv + 2 * o + 2 * h) + (state if case["carried"] else 0), "flops": 14 * n * h * dk * dv}


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_attention(s, train):
    """Token by token: S_t = exp(g_t) S_{t-1} + k_t v_t^T, o_t = scale S_t^T q_t, and the gradients of <o, do> by the
    same recurrence run backwards.  d log decay from the sums of q.dq - k.dk after each token, which 64 bits can take."""
    q, k, v, g = (s[n].detach().double() for n in ("q", "k", "v", "g"))
    group = q.shape[2] // k.shape[2]
    k, v = k.repeat_interleave(group, 2), v.repeat_interleave(group, 2)
    do = s["do"].double() if train else None
    if s["cu"] is not None:
        cu = s["cu"].tolist()
        n, longest, total = len(cu) - 1, s["longest"], q.shape[1]

        def apart(x):
            y = x.new_zeros(n, longest, *x.shape[2:])
            for i in range(n):
                y[i, :cu[i + 1] - cu[i]] = x[0, cu[i]:cu[i + 1]]
            return y

        q, k, v, g = apart(q), apart(k), apart(v), apart(g)
        do = apart(do) if train else None

        def together(x):
            return torch.cat([x[i, :cu[i + 1] - cu[i]] for i in range(n)])[None]
    else:
        def together(x):
            return x
    B, T, H, dk = q.shape
    dv = v.shape[-1]
    a = torch.exp(g)
    S = torch.zeros(B, H, dk, dv, dtype=torch.float64, device=q.device)
    if s["state"] is not None:
        S += s["state"]
    out = torch.empty(B, T, H, dv, dtype=torch.float64, device=q.device)
    dq = torch.empty_like(q)
    for t in range(T):
        S.mul_(a[:, t, :, None, None]).addcmul_(k[:, t, :, :, None], v[:, t, :, None, :])
        out[:, t] = (q[:, t, :, None] @ S)[:, :, 0]
        if train:
            dq[:, t] = (S @ do[:, t, :, :, None])[..., 0]
    out *= s["scale"]
    if not train:
        return {"out": together(out), "state": S}
    dq *= s["scale"]
    R = torch.zeros_like(S)
    dkk, dvv = torch.empty_like(k), torch.empty_like(v)
    for t in range(T - 1, -1, -1):
        R.addcmul_(q[:, t, :, :, None], do[:, t, :, None, :])
        dkk[:, t] = (R @ v[:, t, :, :, None])[..., 0]
        dvv[:, t] = (k[:, t, :, None] @ R)[:, :, 0]
        R.mul_(a[:, t, :, None, None])
    dkk *= s["scale"]
    dvv *= s["scale"]
    dg = ((q * dq).sum(-1) - (k * dkk).sum(-1)).flip(1).cumsum(1).flip(1)
    dkk, dvv = (x.unflatten(2, (-1, group)).sum(3) for x in (dkk, dvv))
    return {"out": together(out), "dq": together(dq), "dk": together(dkk), "dv": together(dvv), "dg": together(dg)}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op.startswith("norm"):
        summed = (s["x"].double() + s["res"].double()).detach()
        h = summed.to(s["res"].dtype).double()  # the norm is that of the sum as it is stored
        w = s["w"].detach().double()
        r = 1.0 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
        y = h * r * w
        if op == "norm":
            return {"y": y, "sum": summed}
        if op == "norm_mxfp8":
            b = y.reshape(y.shape[0], -1, 32)
            e = torch.ceil(torch.log2(b.abs().amax(-1) / 448.0)).clamp(-127, 127)
            scaled = b * torch.pow(2.0, -e)[..., None]
            values = scaled.clamp(-448, 448).to(torch.float8_e4m3fn).double().reshape(y.shape)
            return {"values": values, "scales": torch.pow(2.0, e), "sum": summed}
        dy = s["dy"].double()
        z = dy * w
        dh = r * z - h * r.pow(3) * (z * h).mean(-1, keepdim=True) + s["dsum"].double()
        return {"y": y, "sum": summed, "dx": dh, "dres": dh, "dw": (dy * h * r).sum(0)}
    if op.startswith("rope"):
        rot = case["rot"]
        turn = torch.exp(1j * s["pos"].double()[:, None] * s["freq"]) * s["factor"]

        def rotated(x, turn):
            x = x.detach().double()
            y = x.clone()
            if rot:
                even, odd = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (
                    slice(0, rot // 2), slice(rot // 2, rot))
                z = torch.complex(x[..., even].contiguous(), x[..., odd].contiguous()) * turn[:, None]
                y[..., even], y[..., odd] = z.real, z.imag
            return y

        got = {"q": rotated(s["q"], turn), "k": rotated(s["k"], turn)}
        if op == "rope_train":
            got |= {"dq": rotated(s["dq"], turn.conj()), "dk": rotated(s["dk"], turn.conj())}
        return got
    if op == "step":
        state = s["state"].double()
        out = torch.zeros(*s["q"].shape[:2], case["dv"], dtype=torch.float64, device=state.device)
        group = case["heads"] // case["kv_heads"]
        for i, at in enumerate(s["slots"].tolist()):
            if at < 0:
                continue
            k, v = (s[n][i].double().repeat_interleave(group, 0) for n in ("k", "v"))
            state[at] = state[at] * torch.exp(s["g"][i].double())[:, None, None] + k[:, :, None] * v[:, None, :]
            out[i] = s["scale"] * torch.einsum("hk,hkv->hv", s["q"][i].double(), state[at])
        return {"out": out, "state": state}
    return _exact_attention(s, op == "attn_train")
