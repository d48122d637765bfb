"""Plain 64-bit restatements of the view-token operators on host tensors, with bounds on how far a
kernel's result may be: a rounding to a type is off by half a step (finfo.eps / 2 of the value),
32-bit sums by one 2^-24 of their absolute terms per addition in a chain."""
from __future__ import annotations

import math

import numpy as np
import torch

E32 = 2.0 ** -24  # half a step of a 32-bit float


def half_step(t: torch.dtype) -> float:
    return torch.finfo(t).eps / 2


def tiny(t: torch.dtype) -> float:
    """Half the distance of the type's smallest numbers (16-bit floats lose digits below `tiny`)."""
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


def assert_within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off / bound.clamp(min=1e-300)).nan_to_num(float('inf')).max()):.3g} "
                           f"times the bound; first at {bad.nonzero()[0].tolist()}: {got[bad][0].item()} for {want[bad][0].item()}")


# ---- the generator ----


def philox4x32(counter, key, rounds=10):
    """Philox4x32 on Python's whole numbers (Salmon et al., 2011)."""
    c, k, low = list(counter), list(key), 0xFFFFFFFF
    for _ in range(rounds):
        a, b = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & low, (a >> 32) ^ c[3] ^ k[1], a & low]
        k = [(k[0] + 0x9E3779B9) & low, (k[1] + 0xBB67AE85) & low]
    return c


def keep_mask(n: int, p: float, seed: int, step: int, call: int) -> torch.Tensor:
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    i = np.arange((n + 3) // 4, dtype=np.uint64)
    c = [i & low, i >> u(32), np.full_like(i, u(call)), np.full_like(i, u(step & 0xFFFFFFFF))]
    c = philox4x32_arrays(c, seed)
    words = np.stack(c, -1).reshape(-1)[:n]
    return torch.from_numpy(words >= u(round(p * 2 ** 32)))


def philox4x32_arrays(c, seed):
    u, low = np.uint64, np.uint64(0xFFFFFFFF)
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(10):
        a, b = u(0xD2511F53) * c[0], u(0xCD9E8D57) * c[2]
        c = [(b >> u(32)) ^ c[1] ^ u(k0), b & low, (a >> u(32)) ^ c[3] ^ u(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


# ---- layer norm ----


def layer_norm(z, w, b, eps):
    mu = z.mean(-1, keepdim=True)
    r = 1 / ((z - mu).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (z - mu) * r
    y = xh if w is None else xh * w
    return (y if b is None else y + b), xh, r, mu


def layer_norm_grads(xh, r, dy, w):
    a = dy if w is None else dy * w
    dz = r * (a - a.mean(-1, keepdim=True) - xh * (a * xh).mean(-1, keepdim=True))
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    return dz, flat(dy * xh).sum(0), flat(dy).sum(0)


def norm_noise(z, r, mu):
    """How far xh may be in 32 bits: the mean's and the difference's roundings, scaled by r; the sums over a row are
    chains of width / lanes plus a tree, taken as 64 additions here."""
    return 64 * E32 * (1 + r * (z.abs().amax(-1, keepdim=True) + mu.abs()))


# ---- rotary ----


def rotary(x, positions, freqs, interleaved, factor, back=False):
    """x [B,L,H,D], positions [B,L,A] -> turned, 64 bits"""
    F, A = freqs.numel(), positions.shape[-1]
    angle = torch.stack([positions[..., i // (F // A)].double() * freqs[i] for i in range(F)], -1) if F else positions[..., :0].double()
    c, s = angle.cos()[:, :, None] * factor, angle.sin()[:, :, None] * factor * (-1 if back else 1)
    y = x.clone()
    first, second = (slice(0, 2 * F, 2), slice(1, 2 * F, 2)) if interleaved else (slice(0, F), slice(F, 2 * F))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, a * s + b * c
    return y


# ---- block choice and attention ----


def select_blocks(q, k, top, block, q_lengths=None, kv_lengths=None, allowed=None):
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1:3]
    G, Tq, Tk = Hq // Hkv, -(-Lq // block), -(-Lk // block)
    index = torch.full((B, Hkv, Tq, top), -1, dtype=torch.int32)
    for b in range(B):
        nq = Lq if q_lengths is None else int(q_lengths[b])
        nk = Lk if kv_lengths is None else int(kv_lengths[b])
        for h in range(Hkv):
            km = [k[b, j * block:min(nk, (j + 1) * block), h].mean(0) for j in range(-(-nk // block))]
            for t in range(-(-nq // block)):
                qm = q[b, t * block:min(nq, (t + 1) * block), h * G:(h + 1) * G].mean((0, 1))
                may = [j for j in range(len(km)) if allowed is None or bool(allowed[t, j])]
                best = sorted(may, key=lambda j: (-float((qm * km[j]).sum()), j))[:top]
                index[b, h, t, :len(best)] = torch.tensor(sorted(best), dtype=torch.int32)
    return index


def attention(q, k, v, index, block, q_lengths=None, kv_lengths=None, scale=None, do=None):
    """64-bit inputs -> dict of o (and dq, dk, dv) and *_bound(type) closures' ingredients."""
    B, Lq, Hq, D = q.shape
    Lk, Hkv = k.shape[1:3]
    G, Tk = Hq // Hkv, -(-Lk // block)
    scale = 1 / math.sqrt(D) if scale is None else scale
    see = torch.zeros((B, Hq, Lq, Lk), dtype=torch.bool)
    for b in range(B):
        nq = Lq if q_lengths is None else int(q_lengths[b])
        nk = Lk if kv_lengths is None else int(kv_lengths[b])
        for h in range(Hkv):
            for t in range(index.shape[2]):
                for j in set(index[b, h, t].tolist()):
                    if 0 <= j < Tk:
                        see[b, h * G:(h + 1) * G, t * block:min(nq, (t + 1) * block), j * block:min(nk, (j + 1) * block)] = True
    used = see.any(1).any(1)[:, :, None, None]
    k, v = torch.where(used, k, 0.0), torch.where(used, v, 0.0)  # what nobody sees may be no number
    rows = see.any(-1).permute(0, 2, 1)[..., None]
    q = torch.where(rows, q, 0.0)
    kh, vh = (x.repeat_interleave(G, 2).permute(0, 2, 1, 3) for x in (k, v))
    qh = q.permute(0, 2, 1, 3)
    x = qh @ kh.transpose(-1, -2) * scale
    x = torch.where(see, x, -math.inf)
    p = torch.where(see, torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e300)), 0.0)
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    o = p @ vh
    out = {"o": o.permute(0, 2, 1, 3), "seen": rows}
    n = max(1, int(see.sum(-1).max()))
    xmax = float(torch.where(see, x.abs(), 0.0).max()) if see.any() else 0.0
    # 32 bits: products' sums over D and the keys, the scaled exponent (2^-24 of its value, and of its
    # terms), exp2 itself
    noise = (2 * D + n + 32) * E32 * (1 + xmax + float((qh.abs() @ kh.abs().transpose(-1, -2)).max()) * abs(scale))
    pv = p @ vh.abs()

    def o_bound(t):
        h = half_step(t)  # p is rounded for its product, o at the end
        small = 0.0 if t == torch.float32 else tiny(t) * see.double() @ vh.abs()  # f16: p may be below its normal numbers
        return ((h if t != torch.float32 else 0) * pv + small + h * o.abs() + noise * pv + tiny(t)).permute(0, 2, 1, 3) + 1e-30

    out["o_bound"] = o_bound
    if do is None:
        return out
    do = torch.where(rows, do, 0.0)
    gh = do.permute(0, 2, 1, 3)
    dp = gh @ vh.transpose(-1, -2)
    delta = (gh * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)

    def fold(y):  # [B,Hq,Lk,D] -> [B,Lk,Hkv,D], the shared heads' sum
        return y.unflatten(1, (Hkv, G)).sum(2).permute(0, 2, 1, 3)

    out["dq"] = (ds @ kh * scale).permute(0, 2, 1, 3)
    out["dk"], out["dv"] = fold(ds.transpose(-1, -2) @ qh * scale), fold(p.transpose(-1, -2) @ gh)

    def grads_bound(t):
        h = half_step(t)
        r = h if t != torch.float32 else 0.0
        # f16's smallest numbers: p's as they are, ds's in units of the power of two at the largest |do|
        low = 0.0 if t == torch.float32 else tiny(t) * see.double()
        unit = 2.0 ** math.floor(math.log2(float(do.abs().max()))) if do.abs().max() > 0 else 1.0
        # delta is taken from o as it was rounded; p and ds are rounded for their products; the terms of dp - delta
        # carry 32-bit noise
        e_ds = r * ds.abs() + low * (unit if t == torch.float16 else 1.0) + p * (h * (gh.abs() * o.abs()).sum(-1, keepdim=True)
                                   + noise * (gh.abs() @ vh.abs().transpose(-1, -2) + (gh.abs() * pv).sum(-1, keepdim=True)))
        e_p = r * p + low + noise * p
        rows_n = Lq * G * E32  # chains over the rows
        bq = (e_ds @ kh.abs() * abs(scale)).permute(0, 2, 1, 3) + h * out["dq"].abs() + tiny(t)
        bk = fold((e_ds + rows_n * ds.abs()).transpose(-1, -2) @ qh.abs() * abs(scale)) + h * out["dk"].abs() + tiny(t)
        bv = fold((e_p + rows_n * p).transpose(-1, -2) @ gh.abs()) + h * out["dv"].abs() + tiny(t)
        return tuple(x + 1e-30 for x in (bq, bk, bv))

    out["grads_bound"] = grads_bound
    return out
