"""Operators of the token half of a block, between two channel mixers.

* ``add_rms_norm`` / ``add_rms_norm_mxfp8``: the residual's addition and RMSNorm
  in one pass, with BF16 rows (trains) or MXFP8 rows (serving) out.
* ``rotary_embed`` with ``rotary_frequencies``: rotary positions of queries and
  keys (trains).
* ``linear_attention``: linear attention with a decay per head over batched or
  packed sequences, with carried states (trains); ``linear_attention_step``:
  one token a request against a cache of states.

They run on libspx (``spx_add_rmsnorm_rows``, ``spx_rotary``,
``spx_linear_attention``, ...; ``include/spx.h``) on the current stream of the
tensors' device, without host synchronisation.  The reference's block
(modeling.py:246-302) is where they belong; they restate none of its modules.
"""

from __future__ import annotations

import functools
import math

import torch
from torch import Tensor
from torch.autograd import forward_ad

from spalmer_b200 import _lib
from spalmer_b200.native import _dense

_MAX_HEAD_DIM = 128


_BF16, _F32 = torch.bfloat16, torch.float32
_FLOATS = (_F32, _BF16)
_raw_stream = torch._C._cuda_getCurrentRawStream  # torch.cuda.current_stream(i).cuda_stream without the Stream object
_current_device = torch.cuda.current_device


def _call(name: str, device: torch.device, *args) -> None:
    """Call a libspx entry point on the current stream of ``device`` (which it gets as its last argument)."""

    index = device.index
    fn = getattr(_lib.load(), name)
    if _current_device() == index:
        status = fn(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, _raw_stream(index))
    if status:
        _lib.check(status, name)


def _require(tensor: Tensor, name: str, dtype: torch.dtype | tuple, device: torch.device | None = None) -> None:
    allowed = dtype if isinstance(dtype, tuple) else (dtype,)
    if not isinstance(tensor, Tensor) or not tensor.is_cuda or tensor.dtype not in allowed:
        kinds = " or ".join(str(d).replace("torch.", "") for d in allowed)
        raise ValueError(f"{name} must be a {kinds} CUDA tensor")
    if device is not None and tensor.device != device:
        raise ValueError(f"{name} is on {tensor.device}, not on {device}")


def _refuse_tangents(name: str, *tensors: Tensor | None) -> None:
    """Forward-mode derivatives are not implemented; a dual tensor does not require grad and would lose its tangent."""

    if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{name} has no forward-mode derivative")


def _ptr(t: Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


class _NoSecondDerivative(torch.autograd.Function):
    """The first ``n`` tensors, gradients that depend on the others; a derivative of them raises instead of
    leaving their terms out."""

    @staticmethod
    def forward(ctx, name, n, *tensors):
        ctx.name = name
        return tuple(g.view_as(g) for g in tensors[:n])

    @staticmethod
    def backward(ctx, *_):
        raise NotImplementedError(f"{ctx.name} implements first derivatives only")


def _first_order(name: str):
    """Of an autograd function's backward: it records nothing, and where a graph of it is wanted, that graph raises."""

    def wrap(backward):
        @functools.wraps(backward)
        def wrapped(ctx, *d_outs):
            if not torch.is_grad_enabled():
                return backward(ctx, *d_outs)
            with torch.no_grad():
                out = backward(ctx, *d_outs)
            there = [g for g in out if g is not None]
            needs = [t for t in (*d_outs, *ctx.saved_tensors) if t is not None and t.requires_grad]
            marked = iter(_NoSecondDerivative.apply(name, len(there), *there, *needs) if needs else there)
            return tuple(None if g is None else next(marked) for g in out)
        return wrapped
    return wrap


# ---------------------------------------------------------------- residual + RMSNorm
def _rows(t: Tensor, d: int, item: int) -> Tensor:
    """``t`` as [rows, d] whose rows start on 16 bytes (a copy only if it must be)."""

    if t.is_contiguous():
        r = t.view(-1, d)
        if not r.data_ptr() % 16 and not d * item % 16:
            return r
    else:
        r = t.reshape(-1, d)
    if r.shape[0] and (r.stride(1) != 1 or (r.stride(0) * item) % 16 or r.data_ptr() % 16):
        r = _dense(r)
    return r


def _check_norm(hidden: Tensor, residual: Tensor | None, weight: Tensor, eps: float) -> int:
    _require(hidden, "hidden", torch.bfloat16)
    if hidden.ndim < 1 or hidden.shape[-1] < 1:
        raise ValueError("hidden must be [..., d]")
    d = hidden.shape[-1]
    if residual is not None:
        _require(residual, "residual", (torch.bfloat16, torch.float32), hidden.device)
        if residual.shape != hidden.shape:
            raise ValueError(f"residual must have hidden's shape {tuple(hidden.shape)}")
    _require(weight, "weight", torch.bfloat16, hidden.device)
    if weight.shape != (d,):
        raise ValueError(f"weight must be [{d}]")
    if not eps > 0:
        raise ValueError("eps must be positive")
    return d


def _norm_forward(hidden: Tensor, residual: Tensor | None, weight: Tensor, eps: float, rows: bool,
                  mxfp8: bool) -> tuple[Tensor | None, Tensor | None, Tensor | None, Tensor]:
    """(BF16 rows, MXFP8 values, their scales, sum); sum is hidden itself without a residual."""

    d = hidden.shape[-1]
    x = _rows(hidden, d, 2)
    n, dev = x.shape[0], x.device
    r, f32, total, out, values, scales = None, False, hidden, None, None, None
    if residual is not None:
        f32 = residual.dtype == _F32
        r = _rows(residual, d, 4 if f32 else 2)
        total = torch.empty_like(residual, memory_format=torch.contiguous_format)
    w = _dense(weight) if weight.data_ptr() % 16 or not weight.is_contiguous() else weight
    if rows:
        out = torch.empty_like(hidden, memory_format=torch.contiguous_format)
    if mxfp8:
        values = hidden.new_empty(hidden.shape, dtype=torch.uint8)
        scales = hidden.new_empty((*hidden.shape[:-1], d // 32), dtype=torch.uint8)
    _call("spx_add_rmsnorm_rows", dev, x.data_ptr(), x.stride(0), _ptr(r), 0 if r is None else r.stride(0), f32,
          w.data_ptr(), eps, n, d, None if r is None else total.data_ptr(), _ptr(out), _ptr(values), _ptr(scales))
    return out, values, scales, total


class _AddRMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, hidden, residual, weight, eps):
        out, _, _, total = _norm_forward(hidden, residual, weight, eps, True, False)
        ctx.set_materialize_grads(False)
        ctx.eps = eps
        ctx.has_residual = residual is not None
        ctx.save_for_backward(total, weight)
        if residual is None:
            return out, None
        return out, total

    @staticmethod
    @_first_order("add_rms_norm")
    def backward(ctx, d_out, d_total):
        total, weight = ctx.saved_tensors
        d = weight.shape[0]
        dev = total.device
        if d_out is None:
            d_out = torch.zeros(total.shape, dtype=_BF16, device=dev)
        f32 = total.dtype == _F32
        item = 4 if f32 else 2
        h, dy, w = _rows(total, d, item), _rows(d_out, d, 2), _dense(weight)
        ds = None if d_total is None else _rows(d_total, d, item)
        n = h.shape[0]
        d_hidden = torch.empty_like(d_out, memory_format=torch.contiguous_format)
        d_residual = torch.empty_like(total, memory_format=torch.contiguous_format) if f32 else None
        d_weight = ws = None
        nbytes = 0
        if ctx.needs_input_grad[2]:
            d_weight = torch.empty_like(weight, memory_format=torch.contiguous_format)
            nbytes = _lib.load().spx_add_rmsnorm_backward_workspace(n, d)
            ws = weight.new_empty(nbytes, dtype=torch.uint8)
        _call("spx_add_rmsnorm_backward", dev, h.data_ptr(), h.stride(0), f32, w.data_ptr(), ctx.eps,
              dy.data_ptr(), dy.stride(0), _ptr(ds), 0 if ds is None else ds.stride(0), n, d, d_hidden.data_ptr(),
              _ptr(d_residual), _ptr(d_weight), _ptr(ws), nbytes)
        d_res = None
        if ctx.has_residual:
            d_res = d_residual if f32 else d_hidden  # a BF16 residual's gradient is the same tensor
        return d_hidden, d_res, d_weight, None


def add_rms_norm(hidden: Tensor, residual: Tensor | None, weight: Tensor, eps: float = 1e-6) -> tuple[Tensor, Tensor]:
    """``(normed, summed)``: ``summed = hidden + residual`` in the residual's type and
    RMSNorm of it, ``normed = bf16(summed * weight / sqrt(mean(summed^2) + eps))``.

    ``hidden`` [..., d] BF16, ``residual`` the same shape in BF16 or FP32 (a
    residual stream kept in FP32), ``weight`` [d] BF16; d a multiple of 8 up to
    16,384.  Without a residual ``summed`` is ``hidden`` itself.  Unlike
    ``rms_norm``, which repeats its reference's BF16 roundings in between, the
    result is rounded once.  Differentiable in all three tensors.
    """

    _check_norm(hidden, residual, weight, eps)
    if forward_ad._current_level >= 0:
        _refuse_tangents("add_rms_norm", hidden, residual, weight)
    if torch.is_grad_enabled() and (hidden.requires_grad or weight.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        normed, summed = _AddRMSNorm.apply(hidden, residual, weight, float(eps))
        return normed, hidden if summed is None else summed
    normed, _, _, summed = _norm_forward(hidden, residual, weight, float(eps), True, False)
    return normed, summed


def add_rms_norm_mxfp8(hidden: Tensor, residual: Tensor | None, weight: Tensor, eps: float = 1e-6, *,
                       rows: bool = False) -> tuple[Tensor, ...]:
    """``(values, scales, summed)`` (with ``rows`` the BF16 rows as a fourth): ``add_rms_norm`` with MXFP8 rows out, quantised
    from the FP32 result: E4M3 bytes [..., d] and one E8M0 byte per 32 elements
    [..., d / 32] (uint8), the layout of ``native.mx_quantize_rows`` and the left
    operand of ``native.mxfp8_mm_rows``.  A NaN stays one and has no part in its
    block's scale.  d a multiple of 32.  Forward only.
    """

    d = _check_norm(hidden, residual, weight, eps)
    if d % 32:
        raise ValueError("the row length must be a multiple of the block size 32")
    if forward_ad._current_level >= 0:
        _refuse_tangents("add_rms_norm_mxfp8", hidden, residual, weight)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (hidden, residual, weight)):
        raise NotImplementedError("add_rms_norm_mxfp8 implements the forward pass only")
    normed, values, scales, summed = _norm_forward(hidden, residual, weight, float(eps), rows, True)
    return (values, scales, summed, normed) if rows else (values, scales, summed)


# ---------------------------------------------------------------- rotary positions
def rotary_frequencies(rotary_dim: int, base: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                       original_length: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
                       device: torch.device | str | None = None) -> tuple[Tensor, float]:
    """``(frequencies, factor)`` for ``rotary_embed``: FP64 [rotary_dim / 2] radians per
    position, ``base ** (-2 p / rotary_dim)``, and the factor on sine and cosine (1 unless "yarn").

    ``scaling`` stretches them for contexts ``factor`` times as long as the
    trained ``original_length``: ``"linear"`` divides every frequency,
    ``"ntk"`` raises the base to ``base * factor ** (r / (r - 2))``, and
    ``"yarn"`` divides those that turn less than ``beta_slow`` times over the
    trained length, keeps those that turn more than ``beta_fast`` times, blends
    linearly in between, and scales by ``0.1 ln(factor) + 1``.
    """

    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError("rotary_dim must be even")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError("scaling must be None, 'linear', 'ntk' or 'yarn'")
    if not base > 1 or not factor >= 1 or original_length < 1:
        raise ValueError("base > 1, factor >= 1 and original_length >= 1 are required")
    if scaling == "ntk":
        if rotary_dim < 4:
            raise ValueError("ntk scaling needs rotary_dim >= 4")
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    p = torch.arange(0, rotary_dim, 2, dtype=torch.float64)
    freq = base ** (-p / max(rotary_dim, 1))
    mult = 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        def pair_of(turns: float) -> float:  # the pair that turns `turns` times over the trained length
            return rotary_dim * math.log(original_length / (turns * 2 * math.pi)) / (2 * math.log(base))

        # the ramp may end past the last pair, which after a long trained length still turns more than beta_slow times
        low, high = max(math.floor(pair_of(beta_fast)), 0), min(math.ceil(pair_of(beta_slow)), rotary_dim - 1)
        ramp = ((p / 2 - low) / max(high - low, 1e-3)).clamp(0, 1)
        freq = freq / factor * ramp + freq * (1 - ramp)
        mult = 0.1 * math.log(factor) + 1.0
    return freq.to(device) if device is not None else freq, mult


def _token_heads(t: Tensor) -> Tensor:
    """``t`` [..., heads, d] as [tokens, heads, d] with unit inner stride: a view wherever the leading dimensions merge."""

    if t.stride(-1) != 1 and t.shape[-1] > 1:
        t = t.contiguous()
    return t if t.ndim == 3 else t.reshape(-1, t.shape[-2], t.shape[-1])


def _rotate(q: Tensor, k: Tensor | None, positions: Tensor, frequencies: Tensor, interleaved: bool, factor: float,
            inverse: bool) -> tuple[Tensor, Tensor | None]:
    dev = q.device
    qt = _token_heads(q)
    q_out = torch.empty_like(q, memory_format=torch.contiguous_format)
    n, h, d = qt.shape
    st, sh, _ = qt.stride()
    hq, hk, kt, k_out, kv = _lib.Heads(qt.data_ptr(), 0, st, sh), None, None, None, 0
    if k is not None:
        kt = _token_heads(k)
        k_out = torch.empty_like(k, memory_format=torch.contiguous_format)
        kv = kt.shape[1]
        st, sh, _ = kt.stride()
        hk = _lib.Heads(kt.data_ptr(), 0, st, sh)
    if n:
        pos, freq = positions.contiguous(), frequencies.contiguous()
        _call("spx_rotary", dev, hq, h, hk, kv, n, d, freq.shape[0], pos.data_ptr(), pos.dtype == torch.int64, pos.numel(),
              freq.data_ptr(), factor, interleaved, inverse, q_out.data_ptr(), _ptr(k_out))
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, frequencies, interleaved, factor):
        ctx.save_for_backward(positions, frequencies)
        ctx.args = (interleaved, factor)
        ctx.has_k = k is not None
        return _rotate(q, k, positions, frequencies, interleaved, factor, False)

    @staticmethod
    @_first_order("rotary_embed")
    def backward(ctx, dq, dk):
        positions, frequencies = ctx.saved_tensors
        interleaved, factor = ctx.args
        gq, gk = _rotate(dq, dk if ctx.has_k else None, positions, frequencies, interleaved, factor, True)
        return gq, gk, None, None, None, None


def rotary_embed(q: Tensor, k: Tensor | None, positions: Tensor, frequencies: Tensor, *, interleaved: bool = False,
                 factor: float = 1.0) -> tuple[Tensor, Tensor | None]:
    """Rotary positions: ``(q, k)`` with the first ``2 * len(frequencies)`` elements of
    every head turned by ``position * frequency`` and scaled by ``factor``.

    ``q`` [..., heads, d] and ``k`` [..., kv_heads, d] (or None) BF16, views of a
    fused projection included; ``positions`` int32 or int64, one per token or
    one per token of the last leading dimension (shared by the batch);
    ``frequencies`` FP64 [pairs] (``rotary_frequencies``).  Pairs are halves of
    the rotated part, or neighbours with ``interleaved``.  New contiguous
    tensors come back.  Differentiable in q and k.
    """

    _require(q, "q", torch.bfloat16)
    dev = q.device
    if q.ndim < 3:
        raise ValueError("q must be [..., tokens, heads, head_dim]")
    if k is not None:
        _require(k, "k", torch.bfloat16, dev)
        if k.ndim != q.ndim or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
            raise ValueError("k must be [..., kv_heads, head_dim] over q's tokens")
    _require(positions, "positions", (torch.int32, torch.int64), dev)
    _require(frequencies, "frequencies", torch.float64, dev)
    if frequencies.ndim != 1 or 2 * frequencies.shape[0] > q.shape[-1]:
        raise ValueError("frequencies must be [pairs] with 2 * pairs <= head_dim")
    tokens = math.prod(q.shape[:-2])
    if positions.numel() not in (tokens, q.shape[-3]) or (positions.numel() != tokens and positions.ndim != 1):
        raise ValueError(f"positions must hold one position per token ({tokens}, or {q.shape[-3]} shared by the batch)")
    if forward_ad._current_level >= 0:
        _refuse_tangents("rotary_embed", q, k)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return _Rotary.apply(q, k, positions, frequencies, bool(interleaved), float(factor))
    return _rotate(q, k, positions, frequencies, bool(interleaved), float(factor), False)


# ---------------------------------------------------------------- linear attention
_status: dict[torch.device, int] = {}


def _status_word(device: torch.device) -> int:
    """The address of libspx's status word on ``device``: not memory of PyTorch's, which a graph capture would make its own."""

    word = _status.get(device)
    if word is None:
        at = _lib.ctypes.c_void_p()
        with torch.cuda.device(device):
            _lib.check(_lib.load().spx_token_status_word(at), "spx_token_status_word")
        word = _status[device] = at.value
    return word


def linear_attention_status(device: torch.device | str | int | None = None, clear: bool = True) -> int:
    """The device status word of ``linear_attention`` (synchronises); 0 means no kernel reported an error."""

    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.empty(0, device=device).device
    word = _status.get(dev)
    if word is None:
        return 0
    value = _lib.ctypes.c_int()
    with torch.cuda.device(dev):
        _lib.check(_lib.load().spx_workspace_status(word, value, int(clear), _raw_stream(dev.index)),
                   "spx_workspace_status")
    return value.value


def _aligned_heads(t: Tensor) -> Tensor:
    """``t`` [..., d] (d % 8 == 0) with unit inner stride and rows on 16 bytes (a copy only if it must be)."""

    if t.is_contiguous() and not t.data_ptr() % 16:
        return t
    sizes, strides = t.shape, t.stride()
    if (t.data_ptr() % 16 or strides[-1] != 1
            or any(n > 1 and (st % 8 or st <= 0) for st, n in zip(strides[:-1], sizes[:-1]))):
        t = _dense(t)
    return t


def _heads(t: Tensor) -> _lib.Heads:
    b, n, h, _ = t.stride()
    return _lib.Heads(t.data_ptr(), b, n, h)


def _step_heads(t: Tensor) -> _lib.Heads:
    b, h, _ = t.stride()
    return _lib.Heads(t.data_ptr(), b, 0, h)


def _decays(g: Tensor) -> _lib.Decays:
    return _lib.Decays(g.data_ptr(), *g.stride())


def _dims(q: Tensor, k: Tensor, v: Tensor, g: Tensor, cu: Tensor | None, scale: float) -> _lib.LinAttnDims:
    return _lib.LinAttnDims(q.shape[0] if cu is None else cu.shape[0] - 1, q.shape[1], q.shape[2], k.shape[2],
                            q.shape[3], v.shape[3], int(cu is not None), int(g.dtype == torch.float32), scale)


def _attend(q: Tensor, k: Tensor, v: Tensor, g: Tensor, cu: Tensor | None, state: Tensor | None, scale: float,
            want_state: bool) -> tuple[Tensor, Tensor | None]:
    dev = q.device
    dims = _dims(q, k, v, g, cu, scale)
    out = torch.empty(*q.shape[:3], v.shape[3], dtype=torch.bfloat16, device=dev)
    last = None
    if want_state:
        last = torch.empty(dims.batch, q.shape[2], q.shape[3], v.shape[3], dtype=torch.float32, device=dev)
    nbytes = _lib.load().spx_linear_attention_workspace(dims)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
    _call("spx_linear_attention", dev, dims, _heads(q), _heads(k), _heads(v), _decays(g), _ptr(cu), _ptr(state),
          out.data_ptr(), _ptr(last), _ptr(ws), nbytes, _status_word(dev))
    return out, last


class _LinearAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, state, cu, scale, want_state):
        ctx.set_materialize_grads(False)
        ctx.scale = scale
        ctx.save_for_backward(q, k, v, g, state, cu)
        return _attend(q, k, v, g, cu, state, scale, want_state)

    @staticmethod
    @_first_order("linear_attention")
    def backward(ctx, d_out, d_last):
        q, k, v, g, state, cu = ctx.saved_tensors
        dev = q.device
        dims = _dims(q, k, v, g, cu, ctx.scale)
        if d_out is None:
            d_out = torch.zeros(*q.shape[:3], v.shape[3], dtype=torch.bfloat16, device=dev)
        d_out = _aligned_heads(d_out.to(torch.bfloat16))
        d_last = None if d_last is None else _dense(d_last.float())
        dq, dk, dv = (torch.empty(t.shape, dtype=torch.bfloat16, device=dev) for t in (q, k, v))
        dg = torch.empty(g.shape, dtype=g.dtype, device=dev)
        d_state = torch.empty_like(state) if state is not None and ctx.needs_input_grad[4] else None
        nbytes = _lib.load().spx_linear_attention_backward_workspace(dims)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        _call("spx_linear_attention_backward", dev, dims, _heads(q), _heads(k), _heads(v), _decays(g), _ptr(cu),
              _ptr(state), _heads(d_out), _ptr(d_last), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(),
              _ptr(d_state), _ptr(ws), nbytes, _status_word(dev))
        return dq, dk, dv, dg, d_state, None, None, None


def _check_attention(q: Tensor, k: Tensor, v: Tensor, g: Tensor, scale: float, lead: int, layout: str) -> None:
    _require(q, "q", _BF16)
    dev = q.device
    _require(k, "k", _BF16, dev)
    _require(v, "v", _BF16, dev)
    _require(g, "log_decay", _FLOATS, dev)
    qs, ks, vs = q.shape, k.shape, v.shape
    if len(qs) != lead + 2 or len(ks) != lead + 2 or len(vs) != lead + 2 or g.ndim != lead + 1:
        raise ValueError(f"q, k, v must be [{layout}, heads, dim] and log_decay [{layout}, heads]")
    if ks[:lead] != qs[:lead] or vs[:lead] != qs[:lead] or g.shape != qs[:-1]:
        raise ValueError("q, k, v and log_decay must share their leading dimensions, log_decay q's heads too")
    if ks[-1] != qs[-1] or vs[lead] != ks[lead]:
        raise ValueError("k must have q's head dimension and v the heads of k")
    if ks[lead] < 1 or qs[lead] % ks[lead] or qs[lead] < 1:
        raise ValueError("the query heads must be a multiple of the key/value heads")
    dk, dv = qs[-1], vs[-1]
    if not (8 <= dk <= _MAX_HEAD_DIM and 8 <= dv <= _MAX_HEAD_DIM) or dk % 8 or dv % 8:
        raise ValueError(f"the key and value dimensions of a head must be multiples of 8 up to {_MAX_HEAD_DIM}")
    if not (math.isfinite(scale) and scale != 0):
        raise ValueError("scale must be finite and not zero")


def linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, *, scale: float | None = None,
                     initial_state: Tensor | None = None, cu_seqlens: Tensor | None = None,
                     return_state: bool = False) -> tuple[Tensor, Tensor | None]:
    """Causal linear attention with a decay per head: ``(out, last_state or None)``.

    Per sequence and query head, with the FP32 state S [key_dim, value_dim]:
    ``S_t = exp(log_decay_t) S_{t-1} + k_t v_t^T`` and ``out_t = scale * S_t^T q_t``.

    ``q`` [B, T, heads, key_dim], ``k`` [B, T, kv_heads, key_dim], ``v`` [B, T,
    kv_heads, value_dim] BF16 (views of a fused projection included; query head
    h reads head ``h // (heads // kv_heads)``), ``log_decay`` [B, T, heads]
    FP32 or BF16, natural logarithms meant to be <= 0.  Head dimensions are
    multiples of 8 up to 128; ``scale`` defaults to ``key_dim ** -0.5``.
    ``cu_seqlens`` (int32 [n + 1], within 0 and T, B = 1) packs n sequences into
    one row; tokens before the first offset or after the last (a row padded to a
    fixed length, say) have zero outputs and gradients.  An entry that is out of
    order makes its sequence an empty one and shows in ``linear_attention_status``.  ``initial_state`` and the returned last state
    are FP32 [B or n, heads, key_dim, value_dim].  Nothing passes from one
    sequence to another, non-finite values included; inside one, a value that is
    not finite may reach outputs up to 127 tokens before it.

    Products are summed and states kept in FP32.  In packed rows, and batched ones of
    more than eight tokens, the decayed ``q . k`` and the state are rounded to BF16
    where they are multiplied into ``out`` (2.3e-3 from the exact output in the mean,
    against 1.7e-3 of its own rounding), and into gradients with twice the digits;
    ``out`` may differ in its last bit with ``return_state``, as a state that is
    handed out has FP32's digits.

    Differentiable in q, k, v, log_decay and initial_state, through the output
    and the last state; the backward keeps nothing but the inputs.
    """

    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    _check_attention(q, k, v, log_decay, scale, 2, "batch, tokens")
    dev = q.device
    n = q.shape[0]
    if cu_seqlens is not None:
        _require(cu_seqlens, "cu_seqlens", torch.int32, dev)
        if cu_seqlens.ndim != 1 or cu_seqlens.shape[0] < 1 or q.shape[0] != 1:
            raise ValueError("cu_seqlens must be [sequences + 1] over one packed row (B = 1)")
        cu_seqlens = cu_seqlens.contiguous()
        n = cu_seqlens.shape[0] - 1
    if initial_state is not None:
        _require(initial_state, "initial_state", torch.float32, dev)
        want = (n, q.shape[2], q.shape[3], v.shape[3])
        if tuple(initial_state.shape) != want:
            raise ValueError(f"initial_state must be {list(want)}")
        initial_state = _dense(initial_state)
    if forward_ad._current_level >= 0:
        _refuse_tangents("linear_attention", q, k, v, log_decay, initial_state)
    q, k, v = _aligned_heads(q), _aligned_heads(k), _aligned_heads(v)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (q, k, v, log_decay, initial_state)):
        return _LinearAttention.apply(q, k, v, log_decay, initial_state, cu_seqlens, scale, return_state)
    return _attend(q, k, v, log_decay, cu_seqlens, initial_state, scale, return_state)


def linear_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, *,
                          slots: Tensor | None = None, scale: float | None = None) -> Tensor:
    """One token of each request: updates ``state`` in place, returns ``out`` [B, heads, value_dim].

    ``q`` [B, heads, key_dim], ``k`` and ``v`` [B, kv_heads, ...] BF16,
    ``log_decay`` [B, heads] FP32 or BF16, ``state`` FP32 [slots, heads, key_dim,
    value_dim] contiguous.  Request i uses state ``slots[i]`` (int64 [B]; None:
    i); an index outside the cache (-1, say) marks an empty row, which returns
    zeros and touches nothing.  No index may appear twice.  Forward only.
    """

    scale = float(q.shape[-1] ** -0.5 if scale is None else scale)
    _check_attention(q, k, v, log_decay, scale, 1, "batch")
    dev = q.device
    _require(state, "state", torch.float32, dev)
    B, H, dk = q.shape
    dv = v.shape[-1]
    if state.ndim != 4 or tuple(state.shape[1:]) != (H, dk, dv) or not state.is_contiguous() or state.data_ptr() % 16:
        raise ValueError(f"state must be a contiguous, 16-byte aligned [slots, {H}, {dk}, {dv}]")
    if slots is None:
        if state.shape[0] < B:
            raise ValueError("state holds fewer slots than there are requests")
    else:
        _require(slots, "slots", torch.int64, dev)
        if slots.shape != (B,):
            raise ValueError(f"slots must be [{B}]")
        slots = slots.contiguous()
    if forward_ad._current_level >= 0:
        _refuse_tangents("linear_attention_step", q, k, v, log_decay, state)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or log_decay.requires_grad
                                    or state.requires_grad):
        raise NotImplementedError("linear_attention_step implements the forward pass only")
    q, k, v = _aligned_heads(q), _aligned_heads(k), _aligned_heads(v)
    out = q.new_empty((B, H, dv))
    _call("spx_linear_attention_step", dev, _step_heads(q), _step_heads(k), _step_heads(v),
          _lib.Decays(log_decay.data_ptr(), log_decay.stride(0), 0, log_decay.stride(1)), log_decay.dtype == _F32, B, H,
          k.shape[1], dk, dv, scale, state.data_ptr(), state.shape[0], _ptr(slots), out.data_ptr())
    torch.autograd.graph.increment_version(state)  # written in place: a backward pass that kept it has to notice
    return out


__all__ = [
    "add_rms_norm",
    "add_rms_norm_mxfp8",
    "linear_attention",
    "linear_attention_status",
    "linear_attention_step",
    "rotary_embed",
    "rotary_frequencies",
]
