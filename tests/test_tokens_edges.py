"""View-token operators and their layer at the edges of what they allow."""
from __future__ import annotations

import math

import pytest
import torch

from my_depthsplat_amd import tokens

gpu_only = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


# ---- rows behind the lengths --------------------------------------------------------------


def masked_by_keys(gpu, t, Lq, Lk, Hq, seed):
    """q whose channel 3 is positive, and keys half of which hold -inf there (their score is -inf)."""
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(2, n, h, 32, generator=g) for n, h in ((Lq, Hq), (Lk, 1), (Lk, 1)))
    q[..., 3] = q[..., 3].abs() + 0.5
    k[:, ::2, :, 3] = -math.inf
    return [x.to(gpu, t) for x in (q, k, v)]


@gpu_only
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Lq,Hq,block,blocks,lengths", [(100, 2, 64, 3, (70, 1)), (150, 1, 128, 2, (130, 0)), (64, 1, 32, 5, (33, 31)),
                                                        (5, 4, 64, 40, (3, 1)), (40, 1, 64, 64, (39, 7))])
def test_attention_is_0_behind_the_lengths_whatever_the_keys_hold(gpu, t, Lq, Hq, block, blocks, lengths):
    """Direct and split lists: 0 behind q_lengths beside keys of -inf (a row of zeros times -inf is no number) and values of
    inf; the rows before are the softmax over the other keys."""
    q, k, v = masked_by_keys(gpu, t, Lq, block * blocks - 3, Hq, Lq)
    index = torch.arange(blocks, device=gpu, dtype=torch.int32).expand(2, 1, -(-Lq // block), blocks).contiguous()
    lens = torch.tensor(lengths, device=gpu)
    o = tokens.block_sparse_attention(q, k, v, index, block=block, q_lengths=lens)
    x = (q.double().cpu().transpose(1, 2) @ k[:, 1::2].double().cpu().permute(0, 2, 3, 1)) / 32 ** 0.5
    want = (torch.softmax(x, -1) @ v[:, None, 1::2, 0].double().cpu()).transpose(1, 2)
    # p is rounded to v's type, o too; an exponent's two sums of 32 products are off by 2^-24 * 32 * the products' sizes at most, the sum
    # over the keys by 2^-24 of itself per key of a chain
    big = float((q.abs().max() * k[:, 1::2].abs().max() * 32 / 32 ** 0.5).item())
    bound = (2 * torch.finfo(t).eps / 2 + 2.0 ** -24 * (2 * 32 * big + k.shape[1])) * float(v.abs().max())
    bad = v.clone()
    bad[:, 5] = math.inf
    inf = tokens.block_sparse_attention(q, k, bad, index, block=block, q_lengths=lens)
    for b, n in enumerate(lengths):
        assert float((o[b, :n].double().cpu() - want[b, :n]).abs().amax()) <= bound if n else True
        assert not o[b, n:].any() and not inf[b, n:].any()  # (no number would count)


@gpu_only
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Lq,Hq,block,n", [(100, 2, 64, 70), (150, 1, 128, 130), (64, 1, 32, 33), (130, 3, 64, 65)])
def test_gradients_of_keys_take_nothing_from_rows_behind_the_lengths(gpu, t, Lq, Hq, block, n):
    """dk and dv beside keys of -inf: those of the call that ends at the last row (the same rows in the same units of 32, added in the
    same order)."""
    q, k, v = masked_by_keys(gpu, t, Lq, 3 * block - 3, Hq, Lq)
    index = torch.arange(3, device=gpu, dtype=torch.int32).expand(2, 1, -(-Lq // block), 3).contiguous()
    do = torch.randn(2, Lq, Hq, 32, device=gpu).to(t)
    k.requires_grad_(True), v.requires_grad_(True)
    short = q[:, :n].contiguous()
    want = torch.autograd.grad(tokens.block_sparse_attention(short, k, v, index[:, :, :-(-n // block)].contiguous(), block=block), (k, v), do[:, :n])
    assert all(bool(x.isfinite().all()) and bool((x != 0).any()) for x in want)
    lens = torch.tensor([n, n], device=gpu)
    got = torch.autograd.grad(tokens.block_sparse_attention(q, k, v, index, block=block, q_lengths=lens), (k, v), do)
    for name, a, b in zip(("dk", "dv"), got, want):
        assert torch.equal(a, b), name


@gpu_only
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Lq,blocks", [(1, 1), (1, 5), (1, 9), (1, 17), (7, 33), (70, 6)])
def test_attention_of_infinite_values_in_split_lists(gpu, t, Lq, blocks):
    """A value of inf, in the last block and in the first, is the answer in its channel, and in no other; lists of one part to
    eight."""
    q, k, v = (torch.randn(2, n, h, 32, device=gpu).to(t) for n, h in ((Lq, 2), (blocks * 64, 1), (blocks * 64, 1)))
    v[:, -1, :, 0], v[:, 3, :, 1] = math.inf, -math.inf
    index = torch.arange(blocks, device=gpu, dtype=torch.int32).expand(2, 1, -(-Lq // 64), blocks).contiguous()
    o = tokens.block_sparse_attention(q, k, v, index)
    assert bool((o[..., 0] == math.inf).all()) and bool((o[..., 1] == -math.inf).all()) and bool(o[..., 2:].isfinite().all())
