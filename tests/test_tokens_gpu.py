"""View-token operators on the GPU against their 64-bit restatements (tests/token_oracle.py), whose bounds
count the roundings of the types and of the 32-bit sums."""
from __future__ import annotations

import math

import pytest
import torch

import token_oracle as orc

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
TYPES = [F32, BF16, F16]


def make(gpu, seed):
    g = torch.Generator().manual_seed(seed)

    def rnd(*shape, t=F32, scale=1.0, shift=0.0):
        """(on the GPU in type t, the same values in 64 bits on the host)"""
        x = (torch.randn(shape, generator=g) * scale + shift).to(t)
        return x.to(gpu), x.double()

    return rnd


def tokens():
    from my_depthsplat_amd import tokens as m
    return m


# ---- layer norm -----------------------------------------------------------------------------


def check_norm(gpu, rows, width, t, wt, p=None, mean=0.3, seed=0, use_ds=True, use_dy=True):
    """p None: the plain norm, else the fused form. wt None: no weight, no bias."""
    T = tokens()
    rnd = make(gpu, seed)
    (x, x64), (res, r64) = rnd(rows, width, t=t, scale=1.5, shift=mean), rnd(rows, width, t=t)
    (w, w64), (b, b64) = (rnd(width, t=wt, shift=1.0), rnd(width, t=wt)) if wt is not None else ((None, None),) * 2
    (dy, dy64), (ds, ds64) = rnd(rows, width, t=t), rnd(rows, width, t=t)
    leaves = [v.requires_grad_(True) for v in ((x, res, w, b) if p is not None else (x, w, b)) if v is not None]
    eps, h = 1e-5, orc.half_step(t)
    seed64 = (0x9ABCDEF << 32) | 0x12345678
    if p is None:
        z64, s = x64, None
        y = T.layer_norm(x, w, b, eps)
        drop64 = None
    else:
        rng = T.dropout_rng(seed64, 11, gpu)
        keep = orc.keep_mask(rows * width, p, seed64, 11, 5).view(rows, width)
        scale = 1 / (1 - p) if p < 1 else 0.0
        drop64 = keep.double() * scale
        z64 = torch.where(keep, x64 * scale, 0.0) + r64
        s, y = T.dropout_add_layer_norm(x, res, w, b, p=p, rng=rng, call=5, eps=eps)
        orc.assert_within(s, z64, h * z64.abs() + 3 * orc.E32 * (x64.abs() * scale + r64.abs()) + orc.tiny(t), "s")
        z64 = s.detach().double().cpu()  # the norm is of s as it was rounded
    y64, xh, r, mu = orc.layer_norm(z64, w64, b64, eps)
    wa = 1.0 if w64 is None else w64.abs()
    ba = 0.0 if b64 is None else b64.abs()
    noise = orc.norm_noise(z64, r, mu)
    orc.assert_within(y, y64, h * y64.abs() + noise * (wa * (1 + xh.abs())) + 4 * orc.E32 * ba + orc.tiny(t), "y")
    if not leaves or rows == 0:
        return
    outs, gs = ((y,), (dy,)) if p is None else zip(*([(s, ds)] * use_ds + [(y, dy)] * use_dy))
    got = torch.autograd.grad(outs, leaves, gs, allow_unused=not use_dy)
    d64 = dy64 if use_dy else torch.zeros_like(dy64)
    dz, dw, db = orc.layer_norm_grads(xh, r, d64, w64)
    e = noise * (1 + xh.abs())  # of xh
    a = d64.abs() * wa
    m1, m2 = a.mean(-1, keepdim=True), (a * xh.abs()).mean(-1, keepdim=True)
    ea = (a * e).mean(-1, keepdim=True)
    chain = 64 * orc.E32
    bz = r * (chain * (a + m1 + xh.abs() * m2) + e * m2 + xh.abs() * ea + noise * (a + m1 + xh.abs() * m2))
    want = [dz]
    bound = [bz]
    if p is not None:
        if use_ds:
            dz = dz + ds64
            bz = bz + 2 * orc.E32 * ds64.abs()
        want = [dz * drop64, dz]
        bound = [bz * drop64 + orc.E32 * 2 * (dz * drop64).abs(), bz]
    bound = [v + h * u.abs() + orc.tiny(t) for u, v in zip(want, bound)]
    if wt is not None:
        hw, rows_chain = orc.half_step(wt), (64 + rows / 16) * orc.E32
        want += [dw, db]
        bound += [hw * dw.abs() + (d64.abs() * (e + rows_chain * xh.abs())).sum(0) + orc.tiny(wt),
                  hw * db.abs() + rows_chain * d64.abs().sum(0) + orc.tiny(wt)]
    for name, g, u, v in zip(("dx", "dw", "db") if p is None else ("dx", "dresidual", "dw", "db"), got, want, bound):
        if g is None:
            assert not use_dy and name in ("dw", "db")
            continue
        orc.assert_within(g, u, v, f"{name} {rows}x{width} {t}")


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("width", [1, 2, 3, 4, 7, 8, 9, 31, 64, 100, 127, 128, 129, 250, 513, 768, 1001, 2048, 2051, 4096, 8190, 9001])
def test_layer_norm_widths(gpu, t, width):
    check_norm(gpu, 5 if width > 2000 else 37, width, t, t)


@pytest.mark.parametrize("rows", [0, 1, 2, 63, 4097])
@pytest.mark.parametrize("wt", [None, F32, BF16])
def test_layer_norm_rows_and_weights(gpu, rows, wt):
    check_norm(gpu, rows, 72, BF16, wt, seed=rows)


@pytest.mark.parametrize("mean", [1e4, -3e3])
def test_layer_norm_large_mean(gpu, mean):
    check_norm(gpu, 9, 200, F32, F32, mean=mean)


@pytest.mark.parametrize("t,rows,width,p", [(F32, 33, 128, 0.0), (BF16, 33, 128, 0.3), (F16, 21, 1001, 0.25), (F32, 5, 3, 0.5),
                                            (BF16, 3, 7, 0.5), (F32, 40, 30, 1.0), (F16, 3, 9001, 0.1), (BF16, 3, 5000, 0.1),
                                            (F16, 1, 1, 0.5), (BF16, 300, 770, 0.2)])
def test_dropout_add_layer_norm(gpu, t, rows, width, p):
    check_norm(gpu, rows, width, t, t, p=p)
    check_norm(gpu, rows, width, t, F32, p=p, use_ds=False)
    check_norm(gpu, rows, width, t, None, p=p, use_dy=False)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("width", [6, 96, 1001, 9001])
def test_dropout_add_layer_norm_is_the_two_calls(gpu, t, width):
    T = tokens()
    rng = T.dropout_rng(1, 2, gpu)
    (x, _), (res, _), (w, _), (b, _), (ds, _), (dy, _) = (make(gpu, i)(*s, t=t) for i, s in enumerate([(9, width), (9, width), (width,), (width,), (9, width), (9, width)]))
    leaves = [v.requires_grad_(True) for v in (x, res, w, b)]
    s, y = T.dropout_add_layer_norm(*leaves, p=0.3, rng=rng, call=4)
    s2 = T.dropout(x, 0.3, rng, 4, residual=res)
    y2 = T.layer_norm(s2, w, b)
    assert torch.equal(s, s2) and torch.equal(y, y2)
    got, want = torch.autograd.grad(y, leaves, dy), torch.autograd.grad(y2, leaves, dy)
    assert all(torch.equal(a, c) for a, c in zip(got[2:], want[2:]))
    # the same 32-bit values; where f16's last product and rounding are one instruction it rounds once, else twice
    once = 2 * orc.half_step(F16) * want[1].double().abs() + 2 * orc.tiny(t) if t == F16 else torch.zeros_like(want[1].double())
    assert bool(((got[1].double() - want[1].double()).abs() <= once).all())
    # the two calls round the gradient of s once more before dropout's scale
    both = orc.half_step(t) * (4 + orc.half_step(t)) + 4 * orc.E32
    assert bool(((got[0].double() - want[0].double()).abs() <= both * want[0].double().abs() + 4 * orc.tiny(t)).all())


def test_layer_norm_of_equal_values_and_zero_rows(gpu):
    """Variance 0: y is the bias. Zero rows: empty results, zero weight gradients."""
    T = tokens()
    b = torch.randn(50, device=gpu)
    y = T.layer_norm(torch.full((3, 50), 7.25, device=gpu), None, b)
    assert torch.equal(y, b.expand(3, 50))
    x, w = torch.zeros(0, 50, device=gpu, requires_grad=True), torch.ones(50, device=gpu, requires_grad=True)
    y = T.layer_norm(x, w)
    gx, gw = torch.autograd.grad(y, (x, w), y.detach())
    assert gx.shape == (0, 50) and torch.equal(gw, torch.zeros(50, device=gpu))


def test_layer_norm_of_strided_rows_and_infinite_neighbours(gpu):
    """Rows of another layout give the packed rows' result; a row that is no number touches no other."""
    T = tokens()
    x = torch.randn(6, 40, 9, device=gpu).to(BF16)
    assert torch.equal(T.layer_norm(x.transpose(1, 2)), T.layer_norm(x.transpose(1, 2).contiguous()))
    z = torch.randn(8, 33, device=gpu)
    want = T.layer_norm(z)
    bad = z.clone()
    bad[3, 5], bad[4, 32] = float("inf"), float("nan")
    got = T.layer_norm(bad)
    rows = [0, 1, 2, 5, 6, 7]
    assert torch.equal(got[rows], want[rows]) and got[3:5].isnan().any(1).all()


def test_norm_gradients_are_the_same_bits(gpu):
    T = tokens()
    x = torch.randn(5000, 96, device=gpu).to(BF16).requires_grad_(True)
    w = torch.randn(96, device=gpu, requires_grad=True)
    dy = torch.randn(5000, 96, device=gpu).to(BF16)
    first = torch.autograd.grad(T.layer_norm(x, w), (x, w), dy)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(T.layer_norm(x, w), (x, w), dy)))


# ---- dropout --------------------------------------------------------------------------------


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("n", [1, 3, 4, 5, 8, 11, 1023, 2049, 70001])
def test_dropout_mask_is_the_generators(gpu, t, n):
    T = tokens()
    seed, step, call, p = -3, 2 ** 33 + 9, 77, 0.3
    x, x64 = make(gpu, n)(n, t=t, shift=3.0)
    keep = orc.keep_mask(n, p, seed & (2 ** 64 - 1), step, call)
    y = T.dropout(x, p, T.dropout_rng(seed, step, gpu), call)
    scaled = torch.where(keep, x64 / (1 - p), 0.0)
    orc.assert_within(y, scaled, orc.half_step(t) * scaled.abs() + 3 * orc.E32 * scaled.abs(), "y")
    assert torch.equal((y != 0).cpu(), keep & (x64 != 0))
    res, r64 = make(gpu, n + 1)(n, t=t)
    z = T.dropout(x, p, T.dropout_rng(seed, step, gpu), call, residual=res)
    want = scaled + r64
    orc.assert_within(z, want, orc.half_step(t) * want.abs() + 3 * orc.E32 * (scaled.abs() + r64.abs()) + orc.tiny(t), "y + residual")


def test_dropout_gradients_p0_p1_and_bad_values(gpu):
    T = tokens()
    rng = T.dropout_rng(5, 0, gpu)
    x = torch.randn(3, 50, device=gpu, requires_grad=True)
    res = torch.randn(3, 50, device=gpu, requires_grad=True)
    dy = torch.randn(3, 50, device=gpu)
    keep = orc.keep_mask(150, 0.4, 5, 0, 1).view(3, 50).to(gpu)
    y = T.dropout(x, 0.4, rng, 1, residual=res)
    gx, gr = torch.autograd.grad(y, (x, res), dy)
    torch.testing.assert_close(gx, torch.where(keep, dy / 0.6, 0.0), rtol=4 * orc.E32, atol=0)
    assert torch.equal(gr, dy)
    assert T.dropout(x, 0.0) is x
    assert torch.equal(T.dropout(x, 0.0, residual=res), x + res)
    assert torch.equal(T.dropout(x, 1.0, rng), torch.zeros_like(x))
    assert torch.equal(torch.autograd.grad(T.dropout(x, 1.0, rng), x, dy)[0], torch.zeros_like(x))
    bad = torch.full((3, 50), float("nan"), device=gpu)
    bad[1] = float("inf")
    out = T.dropout(bad, 0.4, rng, 1)
    assert torch.equal(out.isfinite(), ~keep) and bool((out[~keep] == 0).all())
    assert T.dropout(torch.zeros(0, 4, device=gpu), 0.4, rng).shape == (0, 4)


def test_dropout_backward_refuses_a_changed_state(gpu):
    T = tokens()
    rng = T.dropout_rng(5, 0, gpu)
    x = torch.randn(64, device=gpu, requires_grad=True)
    y = T.dropout(x, 0.4, rng)
    rng[1] += 1
    with pytest.raises(RuntimeError):
        y.sum().backward()


def test_dropout_rate_and_independence(gpu):
    """2^20 draws: the kept share is within 5 standard deviations of 1 - p; other calls, steps and seeds keep
    others (their agreement is that of independent masks, within 5 standard deviations)."""
    T = tokens()
    n, p = 1 << 20, 0.25
    one = torch.ones(n, device=gpu)
    masks = [T.dropout(one, p, T.dropout_rng(s, st, gpu), c) != 0 for s, st, c in ((1, 0, 0), (1, 0, 1), (1, 1, 0), (2, 0, 0), (1 + 2 ** 32, 0, 0))]
    for m in masks:
        assert abs(float(m.double().mean()) - (1 - p)) < 5 * math.sqrt(p * (1 - p) / n)
    both = (1 - p) ** 2 + p ** 2
    for m in masks[1:]:
        assert abs(float((m == masks[0]).double().mean()) - both) < 5 * math.sqrt(both * (1 - both) / n)


# ---- rotary ---------------------------------------------------------------------------------


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("B,L,Hq,Hk,D,part,axes,ptype", [
    (2, 5, 3, 1, 64, 64, 1, torch.int64), (1, 1, 8, 2, 128, 64, 1, torch.int32), (3, 7, 2, 2, 24, 12, 2, torch.int64),
    (2, 33, 1, 1, 10, 6, 1, torch.float32), (1, 300, 4, 2, 72, 48, 2, torch.float32), (2, 4, 2, 0, 16, 16, 2, torch.int64),
    (1, 9, 2, 2, 9, 2, 1, torch.int32), (1, 3, 1, 1, 5, 0, 1, torch.int64)])
def test_rotary(gpu, t, inter, B, L, Hq, Hk, D, part, axes, ptype):
    T = tokens()
    rnd = make(gpu, D)
    (q, q64), (dq, dq64) = rnd(B, L, Hq, D, t=t), rnd(B, L, Hq, D, t=t)
    (k, k64), (dk, dk64) = rnd(B, L, max(Hk, 1), D, t=t), rnd(B, L, max(Hk, 1), D, t=t)
    g = torch.Generator().manual_seed(L)
    pos = torch.randint(-5, 2 ** 20, (B, L, axes), generator=g).to(ptype)  # far: 2^20 positions at one radian each
    freqs = T.rotary_frequencies(part, axes, device="cpu") if part else torch.zeros(0, dtype=torch.float64)
    factor = 1.25
    q.requires_grad_(True), k.requires_grad_(True)
    oq, ok = T.rotary(q, k if Hk else None, pos.to(gpu), freqs.to(gpu), interleaved=inter, factor=factor)
    h = orc.half_step(t)

    def bound(x64, want):  # sine and cosine within 4 * 2^-24 of a reduced angle, two products and a sum
        m = (x64.abs().amax(-1, keepdim=True) * factor * 2).expand_as(want)
        return h * want.abs() + 16 * orc.E32 * m + orc.tiny(t)

    for got, x64 in ((oq, q64),) + (((ok, k64),) if Hk else ()):
        want = orc.rotary(x64, pos, freqs, inter, factor)
        orc.assert_within(got, want, bound(x64, want), "turned")
        assert torch.equal(got[..., part:].detach().cpu().double(), x64[..., part:])
    grads = torch.autograd.grad((oq, ok) if Hk else oq, (q, k) if Hk else q, (dq, dk) if Hk else dq)
    for got, x64 in zip(grads, (dq64, dk64)):
        want = orc.rotary(x64, pos, freqs, inter, factor, back=True)
        orc.assert_within(got, want, bound(x64, want), "gradient")


def test_rotary_of_slices(gpu):
    """q and k as strided slices of one projection, positions shared by the batch, broadcast gradients."""
    T = tokens()
    qkv = torch.randn(2, 50, 6, 64, device=gpu).to(BF16).requires_grad_(True)
    pos = T.view_positions(2, 5, 5, gpu)
    fr = T.rotary_frequencies(64, 2, device=gpu)
    q, k = T.rotary(qkv[:, :, :4], qkv[:, :, 4:5], pos, fr)
    packed = [qkv[:, :, :4].detach().contiguous().requires_grad_(True), qkv[:, :, 4:5].detach().contiguous().requires_grad_(True)]
    pq, pk = T.rotary(*packed, pos.expand(2, -1, -1).contiguous(), fr)
    assert torch.equal(q, pq) and torch.equal(k, pk)
    (g,) = torch.autograd.grad(q.float().sum() + 2 * k.float().sum(), qkv)
    one = torch.ones(2, 50, 4, 64, device=gpu, dtype=BF16)
    dq, dk = torch.autograd.grad((pq, pk), packed, (one, 2 * one[:, :, :1].contiguous()))
    assert torch.equal(g, torch.cat([dq, dk, torch.zeros_like(dk)], 2))
    (only,) = torch.autograd.grad(T.rotary(*packed, pos, fr)[1].sum(), packed[1])  # q' unused
    assert only.shape == dk.shape
    (none,) = torch.autograd.grad(T.rotary(packed[0], None, pos, fr)[0], packed[0], one)
    assert torch.equal(none, dq) and T.rotary(packed[0], None, pos, fr)[1] is None


def test_rotary_of_many_sequences(gpu):
    """One token in each of 70001 sequences: the same bits as one sequence of so many tokens."""
    T = tokens()
    q, pos, freqs = torch.randn(70001, 1, 2, 16, device=gpu).to(BF16), torch.arange(70001, device=gpu), T.rotary_frequencies(16, device=gpu)
    got = T.rotary(q, None, pos.view(-1, 1, 1), freqs)[0]
    assert torch.equal(got.view(1, 70001, 2, 16), T.rotary(q.view(1, 70001, 2, 16), None, pos, freqs)[0])


# ---- block choice ---------------------------------------------------------------------------


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("B,Lq,Lk,Hq,Hkv,D,block,top", [
    (2, 70, 200, 4, 2, 16, 32, 3), (1, 1, 1000, 8, 2, 64, 64, 5), (2, 300, 130, 2, 1, 72, 128, 4), (1, 65, 2100, 1, 1, 8, 32, 20),
    (1, 33, 31, 3, 3, 130, 32, 2), (1, 10, 9000, 1, 1, 1, 32, 300), (2, 40, 20001, 2, 1, 12, 32, 7), (1, 33, 66000, 1, 1, 8, 32, 40)])
def test_select_blocks(gpu, t, B, Lq, Lk, Hq, Hkv, D, block, top):
    T = tokens()
    rnd = make(gpu, Lq + Lk)
    (q, q64), (k, k64) = rnd(B, Lq, Hq, D, t=t), rnd(B, Lk, Hkv, D, t=t)
    assert torch.equal(T.select_blocks(q, k, top, block=block).cpu(), orc.select_blocks(q64, k64, top, block))
    g = torch.Generator().manual_seed(1)
    ql, kl = torch.randint(0, Lq + 1, (B,), generator=g), torch.randint(0, Lk + 1, (B,), generator=g)
    may = torch.rand(-(-Lq // block), -(-Lk // block), generator=g) < 0.5
    got = T.select_blocks(q, k, top, block=block, q_lengths=ql.to(gpu), kv_lengths=kl.to(gpu), allowed=may.to(gpu))
    assert torch.equal(got.cpu(), orc.select_blocks(q64, k64, top, block, ql, kl, may))


@pytest.mark.parametrize("blocks", [128, 129, 256, 257, 512, 513, 1024, 1025, 1536, 1537, 2048, 2049])
def test_select_blocks_of_every_number_of_blocks(gpu, blocks):
    """Both sides of each limit between the kernels, with tiles that end inside a group of 16, equal scores and none."""
    T = tokens()
    rnd = make(gpu, blocks)
    Lq, Lk = 18 * 32 + 5, blocks * 32 - 3
    (q, q64), (k, k64) = rnd(2, Lq, 4, 24, t=F16), rnd(2, Lk, 2, 24, t=F16)
    k[:, 32 * 50:32 * 60] = k[:, 32 * 40:32 * 41].repeat(1, 10, 1, 1)
    k64[:, 32 * 50:32 * 60] = k64[:, 32 * 40:32 * 41].repeat(1, 10, 1, 1)
    g = torch.Generator().manual_seed(blocks)
    may = torch.rand(19, blocks, generator=g) < 0.8
    may[3] = False
    ql, kl = torch.tensor([Lq, 260]), torch.tensor([Lk - 40, Lk // 2])
    for top in (1, 16, 200):
        got = T.select_blocks(q, k, top, block=32, q_lengths=ql.to(gpu), kv_lengths=kl.to(gpu), allowed=may.to(gpu))
        assert torch.equal(got.cpu(), orc.select_blocks(q64, k64, top, 32, ql, kl, may))


def test_select_blocks_of_many_rows(gpu):
    """So many rows that few blocks' scores come from the matrix instruction: the same choice as scene by scene."""
    T = tokens()
    q, k = (torch.randn(70, 260 * 32, 1, 128, device=gpu).to(BF16) for _ in range(2))
    k = k[:, :120 * 32]
    got = T.select_blocks(q, k, 6, block=32)
    for b in (0, 33, 69):
        assert torch.equal(got[b:b + 1], T.select_blocks(q[b:b + 1], k[b:b + 1], 6, block=32))


def test_select_blocks_ties_padding_and_no_numbers(gpu):
    """Equal scores go to the lowest blocks, of either sign of zero; rows behind the length do not count, whatever they
    hold; a score that is no number ranks below every other; nothing allowed gives -1."""
    T = tokens()
    k = torch.randn(1, 32, 1, 16, device=gpu).repeat(1, 40, 1, 1)
    q = torch.randn(1, 64, 1, 16, device=gpu)
    assert T.select_blocks(q, k, 5, block=32).flatten().tolist() == [0, 1, 2, 3, 4] * 2
    for blocks in (700, 2100):  # ties and fewer choices than wanted on every path
        k = torch.zeros(1, 32 * blocks, 1, 16, device=gpu)
        k[:, 32 * 5:32 * 6] = q.mean(1, keepdim=True)
        one = q.mean(1, keepdim=True).expand(1, 32, 1, 16)
        assert T.select_blocks(one, k, 4, block=32).flatten().tolist() == [0, 1, 2, 5]
        assert T.select_blocks(-one, -k, 4, block=32).flatten().tolist() == [0, 1, 2, 5]
        may = torch.zeros(1, blocks, dtype=torch.bool, device=gpu)
        may[0, 600], may[0, 650] = True, True
        assert T.select_blocks(one, k, 4, block=32, allowed=may).flatten().tolist() == [600, 650, -1, -1]
    k = torch.randn(1, 320, 1, 16, device=gpu)
    want = T.select_blocks(q[:, :40], k[:, :250], 3, block=32)
    bad_k, bad_q = k.clone(), q.clone()
    bad_k[:, 250:], bad_q[:, 40:] = float("nan"), float("inf")
    lens = dict(q_lengths=torch.tensor([40], device=gpu), kv_lengths=torch.tensor([250], device=gpu, dtype=torch.int32))
    assert torch.equal(T.select_blocks(bad_q, bad_k, 3, block=32, **lens), want)
    nan = k.clone()
    nan[:, 64:96] = float("nan")
    assert not (T.select_blocks(q, nan, 9, block=32) == 2).any()
    assert (T.select_blocks(q, nan, 10, block=32) == torch.arange(10, device=gpu, dtype=torch.int32)).all()
    none = torch.zeros(2, 10, dtype=torch.bool, device=gpu)
    assert (T.select_blocks(q, k, 4, block=32, allowed=none) == -1).all()
    zero = torch.zeros(1, dtype=torch.int32, device=gpu)
    assert (T.select_blocks(q, k, 4, block=32, kv_lengths=zero) == -1).all()
    assert (T.select_blocks(q, k, 4, block=32, q_lengths=zero) == -1).all()
    assert (T.select_blocks(q, k[:, :0], 4, block=32) == -1).all()
    assert T.select_blocks(q[:, :0], k, 4, block=32).shape == (1, 1, 0, 4)


# ---- attention ------------------------------------------------------------------------------


def random_index(B, Hkv, Tq, Tk, top, seed, holes=0.1):
    """Distinct blocks in any order, -1 between them."""
    g = torch.Generator().manual_seed(seed)
    at = torch.rand(B, Hkv, Tq, max(Tk, top), generator=g).argsort(-1)[..., :top]
    at[(at >= Tk) | (torch.rand(at.shape, generator=g) < holes)] = -1
    return at.to(torch.int32)


def check_attention(gpu, t, B, Lq, Lk, Hq, Hkv, D, block, top, lengths=None, index=None, scale=None, train=True, seed=0, spread=1.0):
    T = tokens()
    rnd = make(gpu, seed)
    (q, q64), (k, k64), (v, v64), (do, do64) = (rnd(B, Lq, Hq, D, t=t, scale=spread), rnd(B, Lk, Hkv, D, t=t, scale=spread),
                                                rnd(B, Lk, Hkv, D, t=t), rnd(B, Lq, Hq, D, t=t))
    if index is None:
        index = random_index(B, Hkv, -(-Lq // block), -(-Lk // block), top, seed)
    kw = {} if lengths is None else dict(q_lengths=torch.tensor(lengths[0]), kv_lengths=torch.tensor(lengths[1]))
    want = orc.attention(q64, k64, v64, index, block, scale=scale, do=do64 if train else None, **kw)
    if lengths is not None:  # nothing behind the lengths may matter
        for b in range(B):
            for x, n in ((q, lengths[0]), (do, lengths[0]), (k, lengths[1]), (v, lengths[1])):
                x[b, n[b]:] = float("nan")
    leaves = [x.requires_grad_(train) for x in (q, k, v)]
    o = T.block_sparse_attention(q, k, v, index.to(gpu), block=block, scale=scale, **{n: x.to(gpu) for n, x in kw.items()})
    orc.assert_within(o, want["o"], want["o_bound"](t), f"o {t}")
    if not train:
        return
    bounds = want["grads_bound"](t)
    got = torch.autograd.grad(o, leaves, do)
    for name, g, e in zip(("dq", "dk", "dv"), got, bounds):
        orc.assert_within(g, want[name], e, f"{name} {t}")


SHAPES = [  # B, Lq, Lk, Hq, Hkv, D, block, top
    (1, 64, 64, 1, 1, 64, 64, 1), (2, 200, 300, 2, 1, 64, 64, 3), (1, 130, 513, 4, 2, 32, 32, 5), (1, 257, 257, 1, 1, 128, 64, 4),
    (1, 150, 400, 2, 2, 72, 128, 2), (2, 96, 95, 3, 1, 96, 32, 3), (1, 33, 1, 1, 1, 8, 32, 2), (1, 1, 700, 8, 2, 64, 64, 8),
    (3, 7, 300, 8, 1, 40, 32, 6), (1, 300, 300, 6, 2, 128, 128, 3)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_attention(gpu, t, shape):
    check_attention(gpu, t, *shape, seed=sum(shape))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("block", [32, 64, 128])
def test_attention_of_padded_batches(gpu, t, block):
    """Sequences of other lengths, of none and one among them; what stands behind them is no number."""
    check_attention(gpu, t, 5, 200, 333, 2, 1, 64, block, 3, lengths=([200, 0, 1, 77, 128], [333, 50, 200, 0, 1]), seed=block)


@pytest.mark.parametrize("t", TYPES)
def test_attention_rows_without_blocks_and_places_that_are_none(gpu, t):
    """A tile that chose nothing gives 0 and no gradient; a block named twice counts once; places outside the sequence
    count for nothing."""
    index = torch.tensor([[[[-1, -1, -1, -1], [2, 2, 1, 2], [99, 0, -7, 5], [4, 3, 2 ** 30, 4]]]], dtype=torch.int32)
    check_attention(gpu, t, 1, 128, 160, 2, 1, 32, 32, 4, index=index)


@pytest.mark.parametrize("t", TYPES)
def test_attention_of_large_and_small_scores(gpu, t):
    check_attention(gpu, t, 1, 100, 200, 1, 1, 64, 32, 4, spread=3.0)  # peaked: scores of some tens
    check_attention(gpu, t, 1, 100, 200, 1, 1, 64, 32, 4, scale=0.0)
    check_attention(gpu, t, 1, 100, 200, 1, 1, 64, 32, 4, scale=-0.3)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("block", [32, 128])
def test_attention_of_scores_of_thousands(gpu, t, block):
    check_attention(gpu, t, 1, 200, 300, 2, 1, 64, block, 4, scale=30.0, train=False, seed=block)
    check_attention(gpu, t, 1, 40, 300, 1, 1, 64, block, 4, scale=-300.0, train=False, seed=block)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Lq,Hq,block", [(64, 1, 64), (128, 1, 128), (32, 1, 32), (1, 2, 64), (64, 4, 64)])
def test_attention_of_scores_that_are_minus_infinity(gpu, t, Lq, Hq, block):
    """Keys whose score is -inf count for nothing, wherever in the list they stand: the answer is that of the others, 0
    for a row that has no others. A score of +inf gives no number."""
    T = tokens()
    rnd = make(gpu, block + Lq)
    (q, _), (k, _), (v, _) = rnd(1, Lq, Hq, 32, t=t), rnd(1, 5 * block, 1, 32, t=t), rnd(1, 5 * block, 1, 32, t=t)
    q[..., 3] = q[..., 3].abs() + 0.5
    index = torch.arange(5, device=gpu, dtype=torch.int32).expand(1, 1, 1, 5).contiguous()
    k[:, :block, :, 3] = -float("inf")
    k[:, 2 * block:3 * block - 7, :, 3] = -float("inf")
    keep = k[0, :, 0, 3].isfinite()
    x = torch.einsum("lhd,kd->hlk", q[0].double().cpu(), k[0, :, 0].double().cpu().nan_to_num(neginf=0.0)) / 32 ** 0.5
    p = torch.softmax(x.masked_fill(~keep.cpu(), -float("inf")), -1)
    want = (p @ v[0, :, 0].double().cpu()).transpose(0, 1)[None]
    got = T.block_sparse_attention(q, k, v, index, block=block)
    # p is rounded to v's type, o too; the exponents' sums of 32 products are off by 2^-24 * 32 * max |x| (< 32) at most
    eps = torch.finfo(t).eps / 2
    top = float(v.abs().max())
    assert float((got.double().cpu() - want).abs().max()) <= (2 * eps + 2 * 2.0 ** -24 * 32 * 32) * top
    none = torch.zeros_like(index)
    assert not T.block_sparse_attention(q, k, v, none, block=block).any()
    k[:, 3 * block, :, 3] = float("inf")
    assert T.block_sparse_attention(q, k, v, index, block=block).isnan().all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Lq,Hq,Hkv,B,top", [(1, 8, 2, 3, 40), (1, 1, 1, 1, 60), (5, 4, 1, 2, 33), (40, 1, 1, 1, 64)])
def test_attention_of_few_queries_is_split_and_joined(gpu, t, Lq, Hq, Hkv, B, top):
    check_attention(gpu, t, B, Lq, 64 * 70 - 5, Hq, Hkv, 64, 64, top, seed=top, train=Lq > 1)
    check_attention(gpu, t, B, Lq, 64 * 70 - 5, Hq, Hkv, 64, 64, top, seed=top, train=False,
                    lengths=([Lq] * B, [64 * 70 - 5, 100, 0][:B]))


def test_attention_of_many_tiles_of_one_block(gpu):
    """Every tile chose block 1 (its list spans several words), others chose nothing else."""
    index = torch.full((1, 1, 70, 2), -1, dtype=torch.int32)
    index[..., 1] = 1
    check_attention(gpu, BF16, 1, 70 * 32 - 3, 96, 2, 1, 32, 32, 2, index=index)
    check_attention(gpu, F32, 1, 70 * 32 - 3, 96, 1, 1, 32, 32, 2, index=index)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("block", [32, 64, 128])
def test_attention_of_popular_blocks_in_padded_batches(gpu, t, block):
    """Block 1 is in every tile's list (it is worked off in parts, its rows behind the last key stay 0), block 3 stands
    in half of them twice; the sequences end before, inside and behind them."""
    L, Lk = 40 * block - 3, 4 * block + 5
    index = random_index(3, 2, 40, 5, 4, block, holes=0.5)
    index[..., 1] = 1
    index[..., ::2, 2:] = 3
    check_attention(gpu, t, 3, L, Lk, 4, 2, 40, block, 4, index=index, seed=block,
                    lengths=([L, 1 + L // 3, L - block], [Lk, block - 1, block + 7]))


@pytest.mark.parametrize("t", TYPES)
def test_attention_of_more_blocks_than_workgroups_at_once(gpu, t):
    """Some 1200 key blocks, most of which nobody chose; one is in every list."""
    index = random_index(2, 1, 20, 600, 5, 3)
    index[..., 0] = 7
    check_attention(gpu, t, 2, 20 * 32, 600 * 32 - 9, 2, 1, 24, 32, 5, index=index)


def test_attention_gradients_of_popular_blocks_are_the_same_bits_every_time(gpu):
    T = tokens()
    index = random_index(2, 2, 60, 60, 6, 5).to(gpu)
    index[..., 0] = 11
    q, k, v, do = (torch.randn(2, 60 * 32, h, 64, device=gpu).to(BF16).requires_grad_(True) for h in (4, 2, 2, 4))
    first = None
    for _ in range(5):
        got = torch.autograd.grad(T.block_sparse_attention(q, k, v, index, block=32), (q, k, v), do)
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(got, first))


def test_attention_f16_gradients_far_from_one(gpu):
    """f16 gradients of 2^-12 and 2^8 of the usual size: ds stays within its type's exponents."""
    T = tokens()
    rnd = make(gpu, 3)
    (q, q64), (k, k64), (v, v64), (do, _) = (rnd(1, 64, 1, 32, t=F16) for _ in range(4))
    index = random_index(1, 1, 2, 2, 2, 0, holes=0.0)
    for e in (2.0 ** -12, 2.0 ** 8):
        g = do * e
        want = orc.attention(q64, k64, v64, index, 32, do=g.double().cpu())
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        got = torch.autograd.grad(T.block_sparse_attention(*leaves, index.to(gpu), block=32), leaves, g)
        for name, a, b in zip(("dq", "dk", "dv"), got, want["grads_bound"](F16)):
            orc.assert_within(a, want[name], b, name)


def test_attention_of_slices_and_same_bits(gpu):
    """q, k, v as slices of one projection (strided heads) give the packed tensors' bits, gradients too, every time."""
    T = tokens()
    qkv = torch.randn(2, 150, 8, 64, device=gpu).to(BF16).requires_grad_(True)
    index = random_index(2, 2, 3, 3, 2, 1).to(gpu)
    do = torch.randn(2, 4, 150, 64, device=gpu).to(BF16).transpose(1, 2)
    q, k, v = qkv[:, :, :4], qkv[:, :, 4:6], qkv[:, :, 6:]
    o = T.block_sparse_attention(q, k, v, index)
    packed = [x.detach().contiguous().requires_grad_(True) for x in (q, k, v)]
    op = T.block_sparse_attention(*packed, index)
    assert torch.equal(o, op)
    want = torch.cat(torch.autograd.grad(op, packed, do.contiguous()), 2)
    for _ in range(3):
        (g,) = torch.autograd.grad(T.block_sparse_attention(q, k, v, index), qkv, do)
        assert torch.equal(g, want)


def test_single_tokens_of_any_token_stride(gpu):
    """The stride of a dimension of one token is any number; it is not used."""
    T = tokens()
    any_stride = lambda x: x.as_strided(x.shape, (x.stride(0), 1 << 40, x.stride(2), 1))  # noqa: E731
    q, k, v = (torch.randn(1, 1, h, 16, device=gpu) for h in (4, 2, 2))
    aq, ak, av = (any_stride(x).requires_grad_(True) for x in (q, k, v))
    index = torch.zeros(1, 2, 1, 1, dtype=torch.int32, device=gpu)
    o = T.block_sparse_attention(aq, ak, av, index)
    # One key: o = fl(fl(p v) fl(1 / p)), p = 2^r with the remainder r of the exponent's base, which is rounded: two roundings and a
    # division (within 2.5 units of 2^-23) of v, 7 * 2^-24. Equality held only where r was 0.
    e = 2.0 ** -24
    assert bool(((o - v.repeat_interleave(2, 2)).abs() <= 8 * e * v.repeat_interleave(2, 2).abs()).all())
    grads = torch.autograd.grad(o, (aq, ak, av), any_stride(torch.ones_like(q)))
    # The backward's p = 2^(x - lse): x's two sums of 16 products are off by 16 * 2^-24 of the products' sizes `big` each, lse
    # by a rounding of it and its logarithm's (2 units), exp2 by 2 units; dv is the sum of two such. dp = sum v and delta = sum o
    # are off by 16 * 2^-24 sum |v| each, delta by o's 8 * 2^-24 as well; their difference times the scale of 1 / 4, times k or
    # q (the sum over two heads).
    big = float((q.abs() * k.repeat_interleave(2, 2).abs()).sum(-1).max()) * 0.25 * 1.4427
    assert float((grads[2] - 2.0).abs().max()) <= 2 * e * (2 * 16 * big + big + 16)
    ds = (2 * 16 + 8) * e * float(v.abs().sum(-1).max()) * 1.01
    assert float(grads[0].abs().max()) <= ds / 4 * float(k.abs().max())
    assert float(grads[1].abs().max()) <= 2 * ds / 4 * float(q.abs().max())
    assert torch.equal(T.select_blocks(aq, ak, 1), index)
    pos, freqs = torch.tensor([3], device=gpu), T.rotary_frequencies(16, device=gpu)
    assert all(torch.equal(a, b) for a, b in zip(T.rotary(aq, ak, pos, freqs), T.rotary(q, k, pos, freqs)))


def test_gradients_are_not_differentiable_twice(gpu):
    T = tokens()
    x = torch.randn(4, 8, device=gpu, requires_grad=True)
    (g,) = torch.autograd.grad(T.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_attention_empty_calls(gpu):
    T = tokens()
    z = lambda *s: torch.zeros(*s, device=gpu, requires_grad=True)  # noqa: E731
    i = lambda *s: torch.zeros(*s, device=gpu, dtype=torch.int32)  # noqa: E731
    assert T.block_sparse_attention(z(2, 0, 2, 8), z(2, 5, 1, 8), z(2, 5, 1, 8), i(2, 1, 0, 3)).shape == (2, 0, 2, 8)
    q, k, v = z(2, 5, 2, 8), z(2, 0, 1, 8), z(2, 0, 1, 8)
    o = T.block_sparse_attention(q, k, v, i(2, 1, 1, 3))
    assert torch.equal(o, torch.zeros_like(o))
    assert torch.equal(torch.autograd.grad(o, q, torch.ones_like(o))[0], torch.zeros_like(q))
    q, k, v = z(2, 0, 2, 8), z(2, 5, 1, 8), z(2, 5, 1, 8)
    gk, gv = torch.autograd.grad(T.block_sparse_attention(q, k, v, i(2, 1, 0, 3)), (k, v), torch.zeros(2, 0, 2, 8, device=gpu))
    assert torch.equal(gk, torch.zeros_like(k)) and torch.equal(gv, torch.zeros_like(v))
    assert T.block_sparse_attention(z(0, 5, 2, 8), z(0, 5, 1, 8), z(0, 5, 1, 8), i(0, 1, 1, 3)).shape == (0, 5, 2, 8)
