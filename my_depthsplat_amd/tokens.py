"""Operators of the view-token layer on MI355X: what a transformer over the tokens of all views
needs between the features and the cost volume or the head.

  layer_norm                 rows normalised, scaled and shifted
  dropout                    from a counter-based generator; the mask is never stored
  dropout_add_layer_norm     s = residual + dropout(x), y = layer_norm(s), one pass each way
  rotary                     rotary positions of queries and keys, one or two position axes
  select_blocks              the key blocks each tile of queries attends to
  block_sparse_attention     attention over those blocks
  dropout_rng, rotary_frequencies, view_positions: the inputs they take

float32, bfloat16 or float16 rows; HIP kernels forward and backward (include/dsplat_hip.h, dtk_*;
argument checks and autograd nodes: csrc/dtk_torch.cpp), on torch's current stream of the
tensors' device, without host synchronisation (capturable; a backward pass, as torch has it,
with leaves that no graph made outside the capture holds).
Gradients are the same bits every time (no atomics on them). Not differentiable twice, nor in forward mode (an error).
"""
from __future__ import annotations

import math

import torch

from . import _lib


# ---- layer norm and dropout ---------------------------------------------------------------


def dropout_rng(seed: int, step: int = 0, device="cuda") -> torch.Tensor:
    """The generator's state, int64 [2] = (seed, step) on the device. Calls of one step are told apart
    by their `call` number; advance the step by a new tensor (rng + one) or, once the step's backward
    has run, in place: the backward reads the state again and refuses one that has changed."""
    return torch.tensor([seed, step], dtype=torch.int64, device=device)


def dropout(x: torch.Tensor, p: float, rng: torch.Tensor | None = None, call: int = 0,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """keep * x / (1 - p) (+ residual, of x's shape and type). Element n (row-major) is kept iff word
    n % 4 of Philox4x32-10 of (n / 4, call, step) under the seed is at least p 2^32; rng: dropout_rng().
    A dropped element is 0 whatever it held. p = 0 without a residual returns x."""
    return _lib.load_torch().dropout(x, p, rng, call, residual)


def layer_norm(x: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (biased variance, moments
    in 32 bits). weight, bias [width]: x's type or float32 (both the same), or None."""
    return _lib.load_torch().layer_norm(x, weight, bias, eps)


def dropout_add_layer_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                           bias: torch.Tensor | None = None, p: float = 0.0, rng: torch.Tensor | None = None,
                           call: int = 0, eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """s = residual + dropout(x, p, rng, call), y = layer_norm(s, weight, bias, eps) -> (s, y): the bits
    of the two calls in one pass, and one pass back."""
    return _lib.load_torch().dropout_add_layer_norm(x, residual, weight, bias, p, rng, call, eps)


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


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, freqs: torch.Tensor, *,
           interleaved: bool = False, factor: float = 1.0):
    """Turn pair i of every head by positions[..., axis(i)] * freqs[i], axis(i) = i / (F / axes), times
    `factor` -> (q', k'). q [B,L,Hq,D], k [B,L,Hk,D] or None; positions [L], [L,axes] or [B,L,axes]
    (int64, int32 or float32); freqs float64 [F], 2 F <= D (rotary_frequencies()); pairs (i, i + F), or
    (2i, 2i + 1) if interleaved; the channels behind 2 F stay. Angles are taken in 64 bits. positions and
    freqs have no gradient: those that ask for one are refused."""
    return _lib.load_torch().rotary(q, k, positions, freqs, interleaved, factor)


# ---- attention over chosen blocks ---------------------------------------------------------


def select_blocks(q: torch.Tensor, k: torch.Tensor, top: int, *, block: int = 64, q_lengths: torch.Tensor | None = None,
                  kv_lengths: torch.Tensor | None = None, allowed: torch.Tensor | None = None) -> torch.Tensor:
    """The `top` key blocks of each tile of queries -> int32 [B, Hkv, ceil(Lq / block), top], ascending, -1
    behind. score = (mean query row of the tile, over the heads that share the key head) . (mean key
    row of the block), in 64 bits; ties go to the lowest block. q [B,Lq,Hq,D], k [B,Lk,Hkv,D], D <= 256;
    lengths [B]: rows behind them do not count (None: all do); allowed bool [tiles, blocks] (None:
    all). No gradient: the choice is whole numbers."""
    return _lib.load_torch().select_blocks(q, k, top, block, q_lengths, kv_lengths, allowed)


def block_sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, index: torch.Tensor, *, block: int = 64,
                           q_lengths: torch.Tensor | None = None, kv_lengths: torch.Tensor | None = None,
                           scale: float | None = None) -> torch.Tensor:
    """softmax(scale q k^T) v of the queries of each tile over the keys of its blocks -> [B,Lq,Hq,D].
    q [B,Lq,Hq,D], k, v [B,Lk,Hkv,D] (any strides with dense channels; D a multiple of 8 up to 128; query
    head h reads key head h / (Hq / Hkv), at most 1024 to one); index int32 [B, Hkv, ceil(Lq / block), top <= 1024], as
    select_blocks gives it: places outside the sequence's blocks, and second ones of a block, count
    for nothing. lengths [B] as there: o is 0 behind q_lengths and for queries that see no key. scale (a
    finite number): 1 / sqrt(D) by default. A call that trains in 16 bits takes the probabilities in two pieces
    (its o may differ from a call's without gradients by their rounding) and keeps a second tensor of o's
    size for its backward. Scores and the softmax's statistics are held in 32 bits: past 2^20
    they lose digits that matter, past 2^30 a row may give no number."""
    return _lib.load_torch().block_sparse_attention(q, k, v, index, block, q_lengths, kv_lengths, scale)
