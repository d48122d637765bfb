"""Operators of the view-token layer on MI355X: what a transformer over the tokens of all views
needs between the features and the cost volume or the head.

  layer_norm                 rows normalised, scaled and shifted
  dropout                    from a counter-based generator; the mask is never stored
  dropout_add_layer_norm     s = residual + dropout(x), y = layer_norm(s), one pass each way
  rotary                     rotary positions of queries and keys, one or two position axes
  select_blocks              the key blocks each tile of queries attends to
  block_sparse_attention     attention over those blocks
  dropout_rng, rotary_frequencies, view_positions: the inputs they take

float32, bfloat16 or float16 rows; HIP kernels forward and backward (include/dsplat_hip.h, dtk_*),
on torch's current stream of the tensors' device, without host synchronisation (capturable).
Gradients are the same bits every time (no atomics on them). Not differentiable twice.
"""
from __future__ import annotations

import ctypes
import math

import torch
from torch.autograd.function import once_differentiable

from . import _lib

# the current stream's handle without a Stream object (2 us less per call: a third of a small call's host time)
_raw_stream = torch._C._cuda_getCurrentRawStream

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_POSITION_TYPES = {torch.int64: 4, torch.int32: 3, torch.float32: 0}


def _launch(what: str, dev: torch.device, *args) -> None:
    """lib.what(*args, stream) on torch's current stream of `dev` (kernels are launched on the
    current device, so that is changed where the tensors live elsewhere)."""
    fn = getattr(_lib.load(), what)
    if torch.cuda.current_device() == dev.index:
        status = fn(*args, _raw_stream(dev.index))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, _raw_stream(dev.index))
    if status:
        _lib.check(status, what)


def _same_device(x: torch.Tensor, **others) -> None:
    _lib.require_gpu(x)
    for name, t in others.items():
        if t is not None and t.device != x.device:
            _lib.require_gpu(t)
            raise ValueError(f"{name} is on {t.device}, the rows on {x.device}")


def _row_type(x: torch.Tensor, name: str = "x") -> int:
    if x.dtype not in _TYPES:
        raise ValueError(f"{name} must be float32, bfloat16 or float16, got {x.dtype}")
    return _TYPES[x.dtype]


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _backward(fn):
    """backward() that is not differentiable itself; the wrapper that says so costs 3 us and is left out where
    no graph of the backward is being made."""
    guarded = once_differentiable(fn)

    def backward(ctx, *grads):
        return guarded(ctx, *grads) if torch.is_grad_enabled() else fn(ctx, *grads)

    return staticmethod(backward)


def _contiguous(t):
    return None if t is None else t.contiguous()


# ---- layer norm and dropout ---------------------------------------------------------------


def dropout_rng(seed: int, step: int = 0, device="cuda") -> torch.Tensor:
    """The generator's state, int64 [2] = (seed, step) on the device. Calls of one step are told apart
    by their `call` number; advance the step by a new tensor (rng + one) or, once the step's backward
    has run, in place: the backward reads the state again and refuses one that has changed."""
    return torch.tensor([seed, step], dtype=torch.int64, device=device)


def _check_rng(p: float, rng, call: int) -> float:
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"p must be in [0, 1], got {p}")
    if p > 0.0 and (rng is None or rng.dtype != torch.int64 or rng.numel() != 2 or not rng.is_contiguous()):
        raise ValueError("dropout needs rng, a contiguous int64 tensor (seed, step): dropout_rng()")
    if not 0 <= call < 1 << 32:
        raise ValueError(f"call must be in [0, 2^32), got {call}")
    return p


def _dropout(x, residual, p, rng, call):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _launch("dtk_dropout", x.device, x.numel(), _TYPES[x.dtype], x.data_ptr(), _lib.ptr(residual), p, _lib.ptr(rng), call,
            y.data_ptr())
    return y


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, rng, call):
        ctx.save_for_backward(rng)
        ctx.meta = (p, call)
        return _dropout(x, residual, p, rng, call)

    @_backward
    def backward(ctx, dy):
        (rng,) = ctx.saved_tensors
        p, call = ctx.meta
        dx = _dropout(dy.contiguous(), None, p, rng, call) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor | None = None, call: int = 0,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """keep * x / (1 - p) (+ residual, of x's shape and type). Element n (row-major) is kept iff word
    n % 4 of Philox4x32-10 of (n / 4, call, step) under the seed is at least p 2^32; rng: dropout_rng().
    A dropped element is 0 whatever it held. p = 0 without a residual returns x."""
    p = _check_rng(p, rng, call)
    _row_type(x)
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype):
        raise ValueError(f"residual {residual.dtype} {tuple(residual.shape)} does not match x {x.dtype} {tuple(x.shape)}")
    _same_device(x, residual=residual, rng=rng)
    if p == 0.0 and residual is None:
        return x
    args = (x.contiguous(), _contiguous(residual), p, rng if p > 0.0 else None, call)
    return _Dropout.apply(*args) if _wants_grad(x, residual) else _dropout(*args)


def _norm_fwd(x, residual, weight, bias, eps, p, rng, call, stats):
    width = x.shape[-1]
    rows = x.numel() // width
    s = torch.empty(x.shape, dtype=x.dtype, device=x.device) if residual is not None else None
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    mean = rstd = None
    if stats:
        mean, rstd = torch.empty((2, rows), dtype=torch.float32, device=x.device)
    w = weight if weight is not None else bias
    _launch("dtk_layer_norm_fwd", x.device, rows, width, _TYPES[x.dtype], _TYPES[x.dtype if w is None else w.dtype],
            x.data_ptr(), _lib.ptr(residual), _lib.ptr(weight), _lib.ptr(bias), eps, p, _lib.ptr(rng), call, _lib.ptr(s),
            y.data_ptr(), _lib.ptr(mean), _lib.ptr(rstd))
    return s, y, mean, rstd


def _norm_bwd(z, dy, ds, weight, bias, mean, rstd, add, p, rng, call, needs):
    """needs: of x, residual, weight, bias."""
    width, dev = z.shape[-1], z.device
    rows = z.numel() // width
    if add and p == 0.0 and needs[0] and needs[1]:
        needs = (False, *needs[1:])  # without dropout x's gradient is the residual's
        both = True
    else:
        both = False
    dx, dres = (torch.empty(z.shape, dtype=z.dtype, device=dev) if n else None for n in needs[:2])
    dw, db = (torch.empty(width, dtype=w.dtype, device=dev) if n else None for w, n in zip((weight, bias), needs[2:]))
    ws = None
    if dw is not None or db is not None:
        n = _lib.load().dtk_layer_norm_bwd_workspace_size(rows, width, _TYPES[z.dtype])
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
    w = weight if weight is not None else bias
    _launch("dtk_layer_norm_bwd", dev, rows, width, _TYPES[z.dtype], _TYPES[z.dtype if w is None else w.dtype],
            z.data_ptr(), _lib.ptr(dy), _lib.ptr(ds), _lib.ptr(weight), mean.data_ptr(), rstd.data_ptr(), int(add), p,
            _lib.ptr(rng), call, _lib.ptr(dx), _lib.ptr(dres), _lib.ptr(dw), _lib.ptr(db), _lib.ptr(ws))
    return dres if both else dx, dres, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        _, y, mean, rstd = _norm_fwd(x, None, weight, bias, eps, 0.0, None, 0, True)
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        return y

    @_backward
    def backward(ctx, dy):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        need = ctx.needs_input_grad
        dx, _, dw, db = _norm_bwd(x, dy.contiguous(), None, weight, bias, mean, rstd, False, 0.0, None, 0,
                                  (need[0], False, need[1], need[2]))
        return dx, dw, db, None


class _AddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, p, rng, call):
        s, y, mean, rstd = _norm_fwd(x, residual, weight, bias, eps, p, rng, call, True)
        ctx.save_for_backward(s, weight, bias, mean, rstd, rng)
        ctx.meta = (p, call)
        ctx.set_materialize_grads(False)
        return s, y

    @_backward
    def backward(ctx, ds, dy):
        s, weight, bias, mean, rstd, rng = ctx.saved_tensors
        if ds is None and dy is None:
            return (None,) * 8
        p, call = ctx.meta
        grads = _norm_bwd(s, _contiguous(dy), _contiguous(ds), weight, bias, mean, rstd, True, p, rng, call,
                          ctx.needs_input_grad[:4])
        return (*grads, None, None, None, None)


def _check_norm(x, weight, bias, eps):
    _row_type(x)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"layer norm needs rows [..., width > 0], got {tuple(x.shape)}")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    for name, w in (("weight", weight), ("bias", bias)):
        if w is None:
            continue
        if w.shape != x.shape[-1:]:
            raise ValueError(f"{name} must be [{x.shape[-1]}], got {tuple(w.shape)}")
        if w.dtype not in (x.dtype, torch.float32):
            raise ValueError(f"{name} must be {x.dtype} or float32, got {w.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"weight {weight.dtype} and bias {bias.dtype} must have one type")


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (biased variance, moments
    in 32 bits). weight, bias [width]: x's type or float32 (both the same), or None."""
    _check_norm(x, weight, bias, eps)
    _same_device(x, weight=weight, bias=bias)
    args = (x.contiguous(), _contiguous(weight), _contiguous(bias), float(eps))
    if _wants_grad(x, weight, bias):
        return _LayerNorm.apply(*args)
    return _norm_fwd(args[0], None, *args[1:], 0.0, None, 0, False)[1]


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                           bias: torch.Tensor | None = None, p: float = 0.0, rng: torch.Tensor | None = None,
                           call: int = 0, eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """s = residual + dropout(x, p, rng, call), y = layer_norm(s, weight, bias, eps) -> (s, y): the bits
    of the two calls in one pass, and one pass back."""
    p = _check_rng(p, rng, call)
    _check_norm(x, weight, bias, eps)
    if residual.shape != x.shape or residual.dtype != x.dtype:
        raise ValueError(f"residual {residual.dtype} {tuple(residual.shape)} does not match x {x.dtype} {tuple(x.shape)}")
    _same_device(x, residual=residual, weight=weight, bias=bias, rng=rng)
    args = (x.contiguous(), residual.contiguous(), _contiguous(weight), _contiguous(bias), float(eps), p,
            rng if p > 0.0 else None, call)
    if _wants_grad(x, residual, weight, bias):
        return _AddLayerNorm.apply(*args)
    return _norm_fwd(*args, False)[:2]


# ---- rotary positions ---------------------------------------------------------------------


def rotary_frequencies(part: int, axes: int = 1, base: float = 10000.0, stretch: float = 1.0, trained: int | None = None,
                       device="cuda") -> torch.Tensor:
    """Angle per position of each of the part / 2 pairs, float64 [part / 2]: base^(-i / n) over the n pairs
    of each axis (axis 0's pairs first). stretch > 1 reaches positions that far beyond the trained
    length: without `trained` every pair is slowed down by it; with it only those that turn less than
    once in `trained` positions, those that turn 32 times or more keep their speed, the rest between."""
    if part <= 0 or axes <= 0 or part % (2 * axes):
        raise ValueError(f"part must be a positive multiple of 2 * axes = {2 * axes}, got {part}")
    if not base > 0.0 or not stretch >= 1.0:
        raise ValueError(f"base must be positive and stretch at least 1, got {base} and {stretch}")
    n = part // 2 // axes
    f = base ** (-torch.arange(n, dtype=torch.float64) / n)
    keep = 0.0 if trained is None else ((trained * f / (2 * math.pi) - 1.0) / 31.0).clamp(0.0, 1.0)
    return (f * keep + f / stretch * (1.0 - keep)).repeat(axes).to(device)


def view_positions(views: int, height: int, width: int, device="cuda") -> torch.Tensor:
    """(row, column) of every token of `views` views, int64 [views * height * width, 2]."""
    i = torch.arange(height * width, device=device)
    return torch.stack([i // width, i % width], -1).repeat(views, 1)


def _strides3(t):
    return (ctypes.c_int64 * 3)(*t.stride()[:3])


def _rotary(q, k, positions, freqs, interleaved, factor, back):
    B, L, Hq, D = q.shape
    A = positions.shape[-1]
    ps = positions.stride()
    oq = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ok = None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
    _launch("dtk_rotary", q.device, B, L, Hq, 0 if k is None else k.shape[2], D, freqs.numel(), A, int(interleaved), int(back),
            _TYPES[q.dtype], _POSITION_TYPES[positions.dtype], q.data_ptr(), _strides3(q), _lib.ptr(k),
            None if k is None else _strides3(k), positions.data_ptr(),
            (ctypes.c_int64 * 3)(0 if positions.dim() == 2 else ps[0], ps[-2], ps[-1]), freqs.data_ptr(), factor,
            oq.data_ptr(), _lib.ptr(ok))
    return oq, ok


def _dense_rows(t):
    return t if t.stride(-1) == 1 else t.contiguous()


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, freqs, interleaved, factor):
        ctx.save_for_backward(positions, freqs)
        ctx.meta = (interleaved, factor)
        return _rotary(q, k, positions, freqs, interleaved, factor, False)

    @_backward
    def backward(ctx, dq, dk):
        positions, freqs = ctx.saved_tensors
        dq, dk = _rotary(_dense_rows(dq), None if dk is None else _dense_rows(dk), positions, freqs, *ctx.meta, True)
        return dq, dk, None, None, None, None


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, freqs: torch.Tensor, *,
           interleaved: bool = False, factor: float = 1.0):
    """Turn pair i of every head by positions[..., axis(i)] * freqs[i], axis(i) = i / (F / axes), times
    `factor` -> (q', k'). q [B,L,Hq,D], k [B,L,Hk,D] or None; positions [L], [L,axes] or [B,L,axes]
    (int64, int32 or float32); freqs float64 [F], 2 F <= D (rotary_frequencies()); pairs (i, i + F), or
    (2i, 2i + 1) if interleaved; the channels behind 2 F stay. Angles are taken in 64 bits."""
    if q.dim() != 4 or (k is not None and (k.dim() != 4 or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3])):
        raise ValueError(f"q must be [B,L,Hq,D] and k [B,L,Hk,D], got {tuple(q.shape)}" +
                         ("" if k is None else f" and {tuple(k.shape)}"))
    _row_type(q, "q")
    if k is not None and k.dtype != q.dtype:
        raise ValueError(f"q {q.dtype} and k {k.dtype} must have one type")
    B, L = q.shape[:2]
    if positions.dim() == 1:
        positions = positions[:, None]
    if positions.dim() not in (2, 3) or positions.shape[-2] != L or (positions.dim() == 3 and positions.shape[0] != B):
        raise ValueError(f"positions must be [L={L}], [L,axes] or [B={B},L,axes], got {tuple(positions.shape)}")
    if positions.dtype not in _POSITION_TYPES:
        raise ValueError(f"positions must be int64, int32 or float32, got {positions.dtype}")
    F, axes = freqs.numel(), positions.shape[-1]
    if freqs.dtype != torch.float64 or freqs.dim() != 1 or 2 * F > q.shape[3] or axes == 0 or F % axes:
        raise ValueError(f"freqs must be float64 [F], 2 F <= {q.shape[3]}, F a multiple of the {axes} axes, got "
                         f"{freqs.dtype} {tuple(freqs.shape)}")
    _same_device(q, k=k, positions=positions, freqs=freqs)
    args = (_dense_rows(q), None if k is None else _dense_rows(k), positions, freqs.contiguous(), bool(interleaved),
            float(factor))
    return _Rotary.apply(*args) if _wants_grad(q, k) else _rotary(*args, False)


# ---- attention over chosen blocks ---------------------------------------------------------


def _check_heads(q, k, block, v=None):
    if block not in (32, 64, 128):
        raise ValueError(f"block must be 32, 64 or 128, got {block}")
    if q.dim() != 4 or k.dim() != 4 or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
        raise ValueError(f"q must be [B,Lq,Hq,D] and k [B,Lk,Hkv,D], got {tuple(q.shape)} and {tuple(k.shape)}")
    if k.shape[2] == 0 or q.shape[2] == 0 or q.shape[2] % k.shape[2]:
        raise ValueError(f"the {q.shape[2]} query heads must be a multiple of the {k.shape[2]} key heads")
    if v is not None and v.shape != k.shape:
        raise ValueError(f"v {tuple(v.shape)} does not match k {tuple(k.shape)}")
    _row_type(q, "q")
    if k.dtype != q.dtype or (v is not None and v.dtype != q.dtype):
        raise ValueError("q, k and v must have one type")


def _lengths(t, name, B):
    if t is None:
        return None
    if t.shape != (B,) or t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} must be int32 or int64 [B={B}], got {t.dtype} {tuple(t.shape)}")
    return t


def _int32(t):
    return None if t is None else t.to(torch.int32).contiguous()


def select_blocks(q: torch.Tensor, k: torch.Tensor, top: int, *, block: int = 64, q_lengths: torch.Tensor | None = None,
                  kv_lengths: torch.Tensor | None = None, allowed: torch.Tensor | None = None) -> torch.Tensor:
    """The `top` key blocks of each tile of queries -> int32 [B, Hkv, ceil(Lq / block), top], ascending, -1
    behind. score = (mean query row of the tile, over the heads that share the key head) . (mean key
    row of the block), in 64 bits; ties go to the lowest block. q [B,Lq,Hq,D], k [B,Lk,Hkv,D], D <= 256;
    lengths [B]: rows behind them do not count (None: all do); allowed bool [tiles, blocks] (None:
    all). No gradient: the choice is whole numbers."""
    _check_heads(q, k, block)
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1:3]
    if D > 256 or D == 0:
        raise ValueError(f"the head size must be in [1, 256], got {D}")
    if top <= 0:
        raise ValueError(f"top must be positive, got {top}")
    Tq, Tk = -(-Lq // block), -(-Lk // block)
    q_lengths, kv_lengths = _lengths(q_lengths, "q_lengths", B), _lengths(kv_lengths, "kv_lengths", B)
    if allowed is not None and (allowed.dtype != torch.bool or tuple(allowed.shape) != (Tq, Tk)):
        raise ValueError(f"allowed must be bool [{Tq}, {Tk}], got {allowed.dtype} {tuple(allowed.shape)}")
    _same_device(q, k=k, q_lengths=q_lengths, kv_lengths=kv_lengths, allowed=allowed)
    q, k, allowed = _dense_rows(q.detach()), _dense_rows(k.detach()), _contiguous(allowed)
    q_lengths, kv_lengths = _int32(q_lengths), _int32(kv_lengths)
    index = torch.empty((B, Hkv, Tq, top), dtype=torch.int32, device=q.device)
    ws = torch.empty(_lib.load().dtk_select_blocks_workspace_size(B, Lq, Lk, Hkv, D, block), dtype=torch.uint8,
                     device=q.device)
    _launch("dtk_select_blocks", q.device, B, Lq, Lk, Hq, Hkv, D, block, top, _TYPES[q.dtype], q.data_ptr(), _strides3(q),
            k.data_ptr(), _strides3(k), _lib.ptr(q_lengths), _lib.ptr(kv_lengths), _lib.ptr(allowed), index.data_ptr(),
            ws.data_ptr())
    return index


def _attention(q, k, v, index, block, q_lengths, kv_lengths, scale, o, lse):
    a = _lib.Attention(Lq=q.shape[1], Lk=k.shape[1], B=q.shape[0], Hq=q.shape[2], Hkv=k.shape[2], D=q.shape[3], block=block,
                       top=index.shape[3], dtype=_TYPES[q.dtype], scale=scale, q=q.data_ptr(), k=k.data_ptr(),
                       v=v.data_ptr(), q_strides=q.stride()[:3], k_strides=k.stride()[:3], v_strides=v.stride()[:3],
                       index=index.data_ptr(), q_lengths=_lib.ptr(q_lengths), kv_lengths=_lib.ptr(kv_lengths),
                       o=o.data_ptr(), lse=_lib.ptr(lse))
    return a, ctypes.byref(a)


def _attend(q, k, v, index, block, q_lengths, kv_lengths, scale, stats):
    B, Lq, Hq, D = q.shape
    o = torch.empty((B, Lq, Hq, D), dtype=q.dtype, device=q.device)
    lse = torch.empty((B, Hq, Lq), dtype=torch.float32, device=q.device) if stats else None
    a, ref = _attention(q, k, v, index, block, q_lengths, kv_lengths, scale, o, lse)
    n = _lib.load().dtk_block_sparse_attention_fwd_workspace_size(ref)
    ws = torch.empty(n, dtype=torch.uint8, device=q.device) if n else None
    _launch("dtk_block_sparse_attention_fwd", q.device, ref, _lib.ptr(ws))
    return o, lse


class _Attend(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, index, block, q_lengths, kv_lengths, scale):
        o, lse = _attend(q, k, v, index, block, q_lengths, kv_lengths, scale, True)
        ctx.save_for_backward(q, k, v, index, q_lengths, kv_lengths, o, lse)
        ctx.meta = (block, scale)
        return o

    @_backward
    def backward(ctx, do):
        q, k, v, index, q_lengths, kv_lengths, o, lse = ctx.saved_tensors
        block, scale = ctx.meta
        do = _dense_rows(do)
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        a, ref = _attention(q, k, v, index, block, q_lengths, kv_lengths, scale, o, lse)
        n = _lib.load().dtk_block_sparse_attention_bwd_workspace_size(ref)
        ws = torch.empty(n, dtype=torch.uint8, device=q.device)
        _launch("dtk_block_sparse_attention_bwd", q.device, ref, do.data_ptr(), _strides3(do), dq.data_ptr(), dk.data_ptr(),
                dv.data_ptr(), ws.data_ptr())
        return dq, dk, dv, None, None, None, None, None


def block_sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, index: torch.Tensor, *, block: int = 64,
                           q_lengths: torch.Tensor | None = None, kv_lengths: torch.Tensor | None = None,
                           scale: float | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of the queries of each tile over the keys of its blocks -> [B,Lq,Hq,D].
    q [B,Lq,Hq,D], k, v [B,Lk,Hkv,D] (any strides with dense channels; D a multiple of 8 up to 128; query
    head h reads key head h / (Hq / Hkv)); index int32 [B, Hkv, ceil(Lq / block), top <= 1024], as
    select_blocks gives it: places outside the sequence's blocks, and second ones of a block, count
    for nothing. lengths [B] as there: o is 0 behind q_lengths and for queries that see no key.
    scale: 1 / sqrt(D) by default."""
    _check_heads(q, k, block, v)
    B, Lq, _, D = q.shape
    if D == 0 or D % 8 or D > 128:
        raise ValueError(f"the head size must be a multiple of 8 up to 128, got {D}")
    shape = (B, k.shape[2], -(-Lq // block))
    if index.dtype != torch.int32 or index.dim() != 4 or tuple(index.shape[:3]) != shape or not 1 <= index.shape[3] <= 1024:
        raise ValueError(f"index must be int32 [{shape[0]}, {shape[1]}, {shape[2]}, 1..1024], got {index.dtype} "
                         f"{tuple(index.shape)}")
    q_lengths, kv_lengths = _lengths(q_lengths, "q_lengths", B), _lengths(kv_lengths, "kv_lengths", B)
    _same_device(q, k=k, v=v, index=index, q_lengths=q_lengths, kv_lengths=kv_lengths)
    args = (_dense_rows(q), _dense_rows(k), _dense_rows(v), index.contiguous(), block, _int32(q_lengths), _int32(kv_lengths),
            1.0 / math.sqrt(D) if scale is None else float(scale))
    return _Attend.apply(*args) if _wants_grad(q, k, v) else _attend(*args, False)[0]
