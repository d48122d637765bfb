"""A transformer layer over the tokens of all views of a scene, made of the view-token operators
(tokens.py): what `training.GaussianHead(token_layers=n)` runs between its convolutions.

The reference's multi-view transformer (src/model/encoder/unimatch/mv_transformer.py) attends from every
token to all tokens of the other views; here each tile of 64 tokens attends to the `top` blocks of 64
tokens that a score of their means selects, so the work grows with the number of tokens and not with
its square (12 views of 512 x 960 are 92160 tokens at 1/8).
"""
from __future__ import annotations

import torch
import torch.nn.functional as F
from torch import nn

from . import tokens


class ViewTokenLayer(nn.Module):
    """x [B, L, width] -> the same. y = norm(x); q, k, v of y, q and k turned by (row, column); attention over
    chosen blocks; s = x + dropout(projection), y = norm(s); s + dropout(two-layer network of y).
    heads * 8 must divide width, a head has at most 128 channels; kv_heads (default heads) divides heads."""

    def __init__(self, width: int, heads: int, kv_heads: int | None = None, hidden: int | None = None, top: int = 16,
                 block: int = 64, p: float = 0.0):
        super().__init__()
        kv_heads = heads if kv_heads is None else kv_heads
        if heads <= 0 or width % (8 * heads) or width // heads > 128:
            raise ValueError(f"width {width} must be a multiple of 8 * heads = {8 * heads}, at most 128 per head")
        if kv_heads <= 0 or heads % kv_heads:
            raise ValueError(f"heads {heads} must be a multiple of kv_heads {kv_heads}")
        hidden = 4 * width if hidden is None else hidden
        self.heads, self.kv_heads, self.dim = heads, kv_heads, width // heads
        self.top, self.block, self.p = top, block, p
        self.norm1, self.norm2 = nn.LayerNorm(width), nn.LayerNorm(width)
        self.qkv = nn.Linear(width, (heads + 2 * kv_heads) * self.dim)
        self.out = nn.Linear(width, width)
        self.fc1, self.fc2 = nn.Linear(width, hidden), nn.Linear(hidden, width)

    def part(self, axes: int) -> int:
        """Channels of a head that the positions turn: all that the axes share evenly."""
        return self.dim // (2 * axes) * (2 * axes)

    def forward(self, x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, rng: torch.Tensor | None = None,
                call: int = 0, lengths: torch.Tensor | None = None, allowed: torch.Tensor | None = None) -> torch.Tensor:
        """positions [L, axes] and freqs [part(axes) / 2] as tokens.rotary takes them; rng and call (this layer takes
        two numbers from there) for dropout while training; lengths [B] of a padded batch; allowed
        [tiles, blocks] as tokens.select_blocks takes it."""
        p = self.p if self.training else 0.0
        y = tokens.layer_norm(x, self.norm1.weight, self.norm1.bias, self.norm1.eps)
        qkv = self.qkv(y).unflatten(-1, (-1, self.dim))
        q, k, v = qkv.split((self.heads, self.kv_heads, self.kv_heads), 2)
        q, k = tokens.rotary(q, k, positions, freqs)
        at = dict(block=self.block, q_lengths=lengths, kv_lengths=lengths)
        index = tokens.select_blocks(q, k, self.top, allowed=allowed, **at)
        o = tokens.block_sparse_attention(q, k, v, index, **at)
        # (under autocast the projections come in 16 bits: the sum over the layers stays in the rows' own type)
        s, y = tokens.dropout_add_layer_norm(self.out(o.flatten(2)).to(x.dtype), x, self.norm2.weight, self.norm2.bias, p=p, rng=rng,
                                             call=call, eps=self.norm2.eps)
        return tokens.dropout(self.fc2(F.gelu(self.fc1(y))).to(x.dtype), p, rng, call + 1, residual=s)
