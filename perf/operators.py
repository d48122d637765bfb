"""The view-token operators, measured: layer norm, counter-based dropout, the two fused with the residual sum, rotary
positions, the choice of key blocks, and attention over the chosen blocks.

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()` makes the inputs, `run()` is one pass: the plain
form in elementary torch operations, or the framework's operators where `own` is true. `exact()` is the definition in 64 bits.

Sizes: features of 128 channels at 1/8 resolution (2 views of 256 x 256: 2048 tokens, 6 views of 448 x 768: 32256,
12 views of 512 x 960: 92160), backbone tokens of 768 channels (patches of 14).
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}


def listed():
    return [
        # two 128 x 128 views' features, depth-only inference: the smallest call, latency counts
        dict(name="norm_small", op="norm", dtype="f32", rows=512, width=128, train=False),
        # the backbone tokens of 4 scenes of 6 views of 448 x 768, a training step's norm
        dict(name="norm_backbone_train", op="norm", dtype="bf16", rows=42240, width=768, train=True),
        # dropout + residual + norm with a row length that no vector load divides
        dict(name="add_norm_odd_train", op="add_norm", dtype="f16", rows=20001, width=1001, p=0.25, train=True),
        # the features of two 256 x 256 views
        dict(name="dropout_small_train", op="dropout", dtype="f32", rows=2048, width=128, p=0.1, residual=False, train=True),
        # the hidden rows of the token layer's two-layer network, 4 scenes of 6 views of 448 x 768
        dict(name="dropout_hidden_train", op="dropout", dtype="bf16", rows=129024, width=512, p=0.1, residual=True, train=True),
        # one new token in each of 16 sequences, at a far position, frequencies scaled for it
        dict(name="rotary_one_token", op="rotary", dtype="bf16", batch=16, tokens=1, heads=8, kv_heads=2, dim=64, part=64,
             axes=1, interleaved=False, stretch=8.0, train=False),
        # 12 views of 512 x 960: positions are (row, column) within the view
        dict(name="rotary_12_views_train", op="rotary", dtype="bf16", batch=1, tokens=92160, heads=2, kv_heads=2, dim=64,
             part=64, axes=2, interleaved=True, stretch=1.0, train=True),
        # 4 scenes of 6 views of 448 x 768, blocks of other views only, scenes with fewer tokens among them
        dict(name="select_6_views", op="select", dtype="bf16", batch=4, q_tokens=32256, tokens=32256, heads=2, kv_heads=2,
             dim=64, block=64, top=16, ragged=True, views=6),
        # one new token in each of 16 scenes looks into the scene's tokens
        dict(name="attend_one_token", op="attend", dtype="bf16", batch=16, q_tokens=1, tokens=32256, heads=8, kv_heads=2,
             dim=64, block=64, top=32, ragged=True, train=False),
        # choice and attention of one layer over 12 views of 512 x 960, inference
        dict(name="serve_12_views", op="serve", dtype="bf16", batch=1, q_tokens=92160, tokens=92160, heads=2, kv_heads=2,
             dim=64, block=64, top=16, ragged=False, views=12),
        # 16 scenes of two 256 x 256 views, one head over all channels, 32 bits
        dict(name="attend_2_views_train", op="attend", dtype="f32", batch=16, q_tokens=2048, tokens=2048, heads=1, kv_heads=1,
             dim=128, block=64, top=8, ragged=False, train=True),
        # 4 scenes of 6 views of 448 x 768, two query heads share a key head
        dict(name="attend_6_views_train", op="attend", dtype="bf16", batch=4, q_tokens=32256, tokens=32256, heads=4, kv_heads=2,
             dim=64, block=64, top=16, ragged=True, train=True),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "add_norm", "dropout", "rotary", "select", "attend", "attend", "serve"])
    c = dict(op=op, dtype=rng.choice(["f32", "bf16", "f16"]))
    if op in ("norm", "add_norm", "dropout"):
        c["width"] = _spread(rng, 16, 4096) if rng.random() < 0.5 else 8 * _spread(rng, 4, 256)
        c["rows"] = max(1, min(_spread(rng, 1, 129024), 20_000_000 // c["width"]))
        c["train"] = rng.random() < 0.6
        if op != "norm":
            c["p"] = round(rng.uniform(0.0, 0.6), 3)
        if op == "dropout":
            c["residual"] = rng.random() < 0.5
    elif op == "rotary":
        kv = rng.choice([1, 2, 4])
        c.update(kv_heads=kv, heads=kv * rng.choice([1, 2, 4]), dim=8 * rng.randint(4, 16), batch=rng.randint(1, 8))
        c["tokens"] = max(1, min(_spread(rng, 1, 92160), 24_000_000 // (c["batch"] * c["dim"] * (c["heads"] + kv))))
        c.update(axes=rng.choice([1, 2]), interleaved=rng.random() < 0.5, stretch=rng.choice([1.0, 4.0, 16.0]),
                 train=rng.random() < 0.6)
        c["part"] = 4 * rng.randint(2, c["dim"] // 4)
    else:
        kv = rng.choice([1, 2])
        c.update(kv_heads=kv, heads=kv * rng.choice([1, 2, 4]), dim=8 * rng.randint(4, 16), block=rng.choice([32, 64, 128]),
                 batch=rng.randint(1, 4), top=rng.randint(1, 24), ragged=rng.random() < 0.5)
        c["tokens"] = max(1, min(_spread(rng, 30, 32256), 8_000_000 // (c["batch"] * c["dim"] * c["heads"])))
        c["q_tokens"] = c["tokens"] if rng.random() < 0.6 else rng.choice([1, 7, rng.randint(1, c["tokens"])])
        if op == "attend":
            c["train"] = rng.random() < 0.6
        else:
            c["views"] = 1
    return c


# ---- inputs ---------------------------------------------------------------------------------------------------------


def _frequencies(part, axes, stretch, device):
    """Angle per position of each pair (64 bits): base 10000 over the pairs of one axis; with `stretch` s the pairs that turn
    less than once within 4096 positions are slowed down by s, those that turn 32 times or more are left, the rest between."""
    per = part // 2 // axes
    f = 10000.0 ** (-torch.arange(per, dtype=torch.float64) / per)
    turns = 4096.0 * f / (2 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0, 1)
    return (f * keep + f / stretch * (1 - keep)).repeat(axes).to(device)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=g, device=dev) * scale + shift).to(t)

    op, s = case["op"], {"case": case}
    if op in ("norm", "add_norm", "dropout"):
        n, c = case["rows"], case["width"]
        s["x"] = normal(n, c, scale=1.5, shift=0.3)
        if op == "add_norm" or case.get("residual"):
            s["residual"] = normal(n, c)
        if op != "dropout":
            s["weight"], s["bias"] = normal(c, scale=0.2, shift=1.0), normal(c, scale=0.1)
        if op != "norm":
            s["rng"] = torch.tensor([seed * 7919 + 12345678901, seed % 1000 + 3], dtype=torch.int64, device=dev)
        if case["train"]:
            s["dy"] = normal(n, c)
            if op == "add_norm":
                s["ds"] = normal(n, c)
    elif op == "rotary":
        b, l, d = case["batch"], case["tokens"], case["dim"]
        s["q"], s["k"] = normal(b, l, case["heads"], d), normal(b, l, case["kv_heads"], d)
        if case["axes"] == 2:  # (row, column) of a token in a view about 1.8 times as wide as high
            w = max(1, int(math.sqrt(1.8 * min(l, 7680))))
            i = torch.arange(l, device=dev) % 7680
            s["positions"] = torch.stack([i // w, i % w], -1).expand(b, l, 2).contiguous()
        else:  # sequences of another length so far
            at = torch.randint(0, 30000, (b, 1), generator=g, device=dev)
            s["positions"] = (at + torch.arange(l, device=dev))[..., None].contiguous()
        s["freqs"] = _frequencies(case["part"] - case["part"] % (2 * case["axes"]), case["axes"], case["stretch"], dev)
        if case["train"]:
            s["dq"], s["dk"] = normal(*s["q"].shape), normal(*s["k"].shape)
    else:
        b, lq, l, h, kv, d = (case[n] for n in ("batch", "q_tokens", "tokens", "heads", "kv_heads", "dim"))
        block = case["block"]
        tq, tk = -(-lq // block), -(-l // block)
        # tokens of one block resemble each other, and blocks of other views that show the same place
        place = torch.randn((b, tk, kv, d), generator=g, device=dev) * 0.6
        place = place.repeat_interleave(block, 1)[:, :l]
        s["k"] = (torch.randn((b, l, kv, d), generator=g, device=dev) * 0.8 + place).to(t)
        s["v"] = normal(b, l, kv, d)
        q = torch.randn((b, lq, h, d), generator=g, device=dev) * 0.8
        q = q + place[:, torch.arange(lq, device=dev) * l // lq].roll(l // 7, 1).repeat_interleave(h // kv, 2)
        s["q"] = q.to(t)
        s["q_lengths"] = s["kv_lengths"] = None
        if case["ragged"]:  # a padded batch: some sequences are shorter
            s["kv_lengths"] = torch.randint(l // 2, l + 1, (b,), generator=g, device=dev, dtype=torch.int32)
            s["q_lengths"] = torch.randint(max(1, lq // 2), lq + 1, (b,), generator=g, device=dev, dtype=torch.int32)
        if op in ("select", "serve"):
            s["allowed"] = None
            if case["views"] > 1:  # other views' blocks only
                view = torch.arange(tk, device=dev) * case["views"] // tk
                s["allowed"] = view[:tq, None] != view[None]
        else:  # a chosen index: some blocks are popular, some tiles have chosen fewer
            like = torch.rand((b, kv, 1, tk), generator=g, device=dev) * 0.4 + torch.rand((b, kv, tq, tk), generator=g, device=dev)
            n = min(case["top"], tk)
            at = like.topk(n, -1).indices
            at = torch.nn.functional.pad(at, (0, case["top"] - n), value=tk)
            few = torch.rand((b, kv, tq, case["top"]), generator=g, device=dev) < 0.03
            at = at.masked_fill(few, tk).sort(-1).values
            s["index"] = at.masked_fill(at == tk, -1).to(torch.int32)
            if case["train"]:
                s["do"] = normal(b, lq, h, d)
    if case.get("train"):
        for n in ("x", "residual", "weight", "bias", "q", "k", "v"):
            if n in s:
                s[n].requires_grad_(True)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return _PLAIN[s["case"]["op"]](s, s["case"])


def _run_own(s):
    from my_depthsplat_amd import tokens
    c = s["case"]
    op, train = c["op"], c.get("train")
    if op == "norm":
        y = tokens.layer_norm(s["x"], s["weight"], s["bias"])
        return {"y": y, "grads": torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["dy"])} if train else {"y": y}
    if op == "add_norm":
        z, y = tokens.dropout_add_layer_norm(s["x"], s["residual"], s["weight"], s["bias"], p=c["p"], rng=s["rng"], call=1)
        out = {"s": z, "y": y}
        if train:
            leaves = (s["x"], s["residual"], s["weight"], s["bias"])
            out["grads"] = torch.autograd.grad((z, y), leaves, (s["ds"], s["dy"]))
        return out
    if op == "dropout":
        y = tokens.dropout(s["x"], c["p"], s["rng"], call=2, residual=s.get("residual"))
        if not train:
            return {"y": y}
        leaves = (s["x"], s["residual"]) if c["residual"] else (s["x"],)
        return {"y": y, "grads": torch.autograd.grad(y, leaves, s["dy"])}
    if op == "rotary":
        q, k = tokens.rotary(s["q"], s["k"], s["positions"], s["freqs"], interleaved=c["interleaved"])
        out = {"q": q, "k": k}
        if train:
            out["grads"] = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return out
    lengths = dict(q_lengths=s["q_lengths"], kv_lengths=s["kv_lengths"])
    if op in ("select", "serve"):
        index = tokens.select_blocks(s["q"], s["k"], c["top"], block=c["block"], allowed=s["allowed"], **lengths)
        if op == "select":
            return {"index": index}
        return {"index": index, "o": tokens.block_sparse_attention(s["q"], s["k"], s["v"], index, block=c["block"], **lengths)}
    o = tokens.block_sparse_attention(s["q"], s["k"], s["v"], s["index"], block=c["block"], **lengths)
    return {"o": o, "grads": torch.autograd.grad(o, (s["q"], s["k"], s["v"]), s["do"])} if train else {"o": o}


def _norm_backward(xh, r, dy, w, t):
    """(gradient of the rows in 32 bits, of the weight, of the bias)"""
    dxh = dy * w
    dx = r * (dxh - dxh.mean(-1, keepdim=True) - xh * (dxh * xh).mean(-1, keepdim=True))
    return dx, (dy * xh).sum(0).to(t), dy.sum(0).to(t)


def _normalise(x):
    x = x - x.mean(-1, keepdim=True)
    r = (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    return x * r, r


def _plain_norm(s, c):
    t = s["x"].dtype
    w, b = s["weight"].float(), s["bias"].float()
    xh, r = _normalise(s["x"].float())
    y = (xh * w + b).to(t)
    if not c["train"]:
        return {"y": y}
    dx, dw, db = _norm_backward(xh, r, s["dy"].float(), w, t)
    return {"y": y, "grads": (dx.to(t), dw, db)}


def _keep(shape, p, rng, call):
    """Which elements dropout keeps. Element n takes word n % 4 of Philox4x32-10 (Salmon et al., Parallel random numbers: as
    easy as 1, 2, 3, 2011) of the counter (n / 4 in two words, call, step) under the key (seed in two words)."""
    n = math.prod(shape)
    low = 0xFFFFFFFF
    i = torch.arange((n + 3) // 4, device=rng.device)
    c = [i & low, i >> 32, torch.full_like(i, call), (rng[1] & low).expand_as(i)]
    k0, k1 = rng[0] & low, (rng[0] >> 32) & low
    for r in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57  # 64-bit products, the sign bit is the highest of the upper word
        c = [((b >> 32) & low) ^ c[1] ^ k0, b & low, ((a >> 32) & low) ^ c[3] ^ k1, a & low]
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack(c, -1).reshape(-1)[:n].reshape(shape) >= round(p * 2.0 ** 32)


def _plain_dropout(s, c):
    x, t = s["x"].float(), s["x"].dtype
    keep = _keep(x.shape, c["p"], s["rng"], 2)
    y = torch.where(keep, x * (1 / (1 - c["p"])), 0.0)
    if c["residual"]:
        y = y + s["residual"].float()
    if not c["train"]:
        return {"y": y.to(t)}
    dx = torch.where(keep, s["dy"].float() * (1 / (1 - c["p"])), 0.0).to(t)
    return {"y": y.to(t), "grads": (dx, s["dy"]) if c["residual"] else (dx,)}


def _plain_add_norm(s, c):
    x, t = s["x"].float(), s["x"].dtype
    keep = _keep(x.shape, c["p"], s["rng"], 1)
    z = s["residual"].float() + torch.where(keep, x * (1 / (1 - c["p"])), 0.0)
    w, b = s["weight"].float(), s["bias"].float()
    xh, r = _normalise(z)
    out = {"s": z.to(t), "y": (xh * w + b).to(t)}
    if c["train"]:
        dz, dw, db = _norm_backward(xh, r, s["dy"].float(), w, t)
        dz = dz + s["ds"].float()
        out["grads"] = (torch.where(keep, dz * (1 / (1 - c["p"])), 0.0).to(t), dz.to(t), dw, db)
    return out


def _turn(x, cos, sin, interleaved):
    t, x, n = x.dtype, x.float(), cos.shape[-1]
    if interleaved:
        a, b = x[..., 0:2 * n:2], x[..., 1:2 * n:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    else:
        a, b = x[..., :n], x[..., n:2 * n]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, x[..., 2 * n:]], -1).to(t)


def _plain_rotary(s, c):
    n = s["freqs"].numel() // c["axes"]
    angle = s["positions"].double().repeat_interleave(n, -1) * s["freqs"]  # far positions: in 64 bits
    cos, sin = (f(angle).float()[:, :, None] for f in (torch.cos, torch.sin))
    out = {n: _turn(s[n], cos, sin, c["interleaved"]) for n in ("q", "k")}
    if c["train"]:
        out["grads"] = tuple(_turn(s[n], cos, -sin, c["interleaved"]) for n in ("dq", "dk"))
    return out


def _tiles(x, block, lengths, t):
    """[B, L, H, D] -> [B, H, tiles, block, D] with zeros behind each sequence's length, and which rows count [B, tiles, block]"""
    b, l = x.shape[:2]
    n = -(-l // block)
    at = torch.arange(n * block, device=x.device)
    valid = at < (l if lengths is None else lengths.clamp(max=l)[:, None])
    valid = valid.expand(b, -1)
    x = torch.nn.functional.pad(x.to(t), (0, 0, 0, 0, 0, n * block - l))
    x = torch.where(valid[..., None, None], x, 0.0)
    return x.permute(0, 2, 1, 3).unflatten(2, (n, block)), valid.unflatten(1, (n, block))


def _plain_select(s, c):
    b, kv, top = c["batch"], c["kv_heads"], c["top"]
    q, qv = _tiles(s["q"], c["block"], s["q_lengths"], torch.float64)  # in 64 bits: near scores, and whole numbers come out
    k, kvd = _tiles(s["k"], c["block"], s["kv_lengths"], torch.float64)
    qm = q.sum(3).unflatten(1, (kv, -1)).sum(2) / (qv.sum(-1)[:, None, :, None] * (c["heads"] // kv)).clamp(min=1)
    km = k.sum(3) / kvd.sum(-1)[:, None, :, None].clamp(min=1)
    score = torch.matmul(qm, km.transpose(-1, -2))
    may = (qv.any(-1)[:, None, :, None] & kvd.any(-1)[:, None, None, :]).expand(score.shape)
    if s["allowed"] is not None:
        may = may & s["allowed"]
    tk = score.shape[-1]
    at = torch.sort(torch.where(may, score, -math.inf), dim=-1, descending=True, stable=True).indices[..., :top]
    at = torch.where(may.gather(-1, at), at, tk).sort(-1).values
    at = torch.nn.functional.pad(at, (0, top - at.shape[-1]), value=tk)
    return {"index": torch.where(at == tk, -1, at).to(torch.int32)}


def _chosen(x, index):
    """[B, Hkv, blocks, block, D], [B, Hkv, tiles, top] -> [B, Hkv, tiles, top * block, D]"""
    b, h = index.shape[:2]
    ib, ih = torch.arange(b, device=x.device)[:, None, None, None], torch.arange(h, device=x.device)[:, None, None]
    return x[ib, ih, index].flatten(3, 4)


def _plain_attend(s, c):
    b, lq, l, h, kv, d, block = (c[n] for n in ("batch", "q_tokens", "tokens", "heads", "kv_heads", "dim", "block"))
    t, scale = s["q"].dtype, 1 / math.sqrt(c["dim"])

    def rows(x):  # [B, L, H, D] -> [B, Hkv, tiles, group * block, D]
        x, _ = _tiles(x, block, s["q_lengths"], torch.float32)
        return x.unflatten(1, (kv, h // kv)).transpose(2, 3).flatten(3, 4)

    def back(x, n):  # the other way, to n tokens
        x = x.unflatten(3, (-1, block)).transpose(2, 3).flatten(1, 2).flatten(2, 3)
        return x[:, :, :n].transpose(1, 2).to(t)

    q = rows(s["q"])
    k, valid = _tiles(s["k"], block, s["kv_lengths"], torch.float32)
    v, _ = _tiles(s["v"], block, s["kv_lengths"], torch.float32)
    index = s["index"].clamp(min=0).long()
    kc, vc = _chosen(k, index), _chosen(v, index)
    see = valid[torch.arange(b, device=k.device)[:, None, None, None], index] & (s["index"] >= 0)[..., None]
    see = see.flatten(3, 4)[..., None, :]
    x = torch.where(see, torch.matmul(q, kc.transpose(-1, -2)) * scale, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-30)
    inside = _tiles(torch.ones_like(s["q"][:, :, :1, :1]), block, s["q_lengths"], torch.float32)[0]  # [B, 1, tiles, block, 1]
    inside = inside.repeat(1, 1, 1, h // kv, 1)
    o = torch.matmul(p, vc) * inside
    out = {"o": back(o, lq)}
    if c.get("train"):
        do = rows(s["do"])
        dx = p * (torch.matmul(do, vc.transpose(-1, -2)) - (do * o).sum(-1, keepdim=True)) * scale
        dq = torch.matmul(dx, kc)
        dk, dv = torch.matmul(dx.transpose(-1, -2), q), torch.matmul(p.transpose(-1, -2), do)
        n = k.shape[2]
        at = ((torch.arange(b, device=k.device)[:, None] * kv + torch.arange(kv, device=k.device))[..., None, None] * n + index)
        g = [torch.zeros((b * kv * n, block * d), device=k.device).index_add_(0, at.flatten(), e.reshape(-1, block * d))
             for e in (dk, dv)]
        g = [e.reshape(b, kv, n * block, d)[:, :, :l].transpose(1, 2).to(t) for e in g]
        out["grads"] = (back(dq, lq), g[0], g[1])
    return out


def _plain_serve(s, c):
    index = _plain_select(s, c)["index"]
    return {"index": index, "o": _plain_attend({**s, "index": index}, c)["o"]}


_PLAIN = {"norm": _plain_norm, "add_norm": _plain_add_norm, "dropout": _plain_dropout, "rotary": _plain_rotary,
          "select": _plain_select, "attend": _plain_attend, "serve": _plain_serve}


# ---- what a pass cannot do without ----------------------------------------------------------------------------------


def work(c):
    e = SIZE[c["dtype"]]
    op, train = c["op"], c.get("train", False)
    if op in ("norm", "add_norm", "dropout"):
        n = c["rows"] * c["width"]
        if op == "norm":  # x -> y; x, dy -> dx
            return {"bytes": n * e * (5 if train else 2), "flops": n * (20 if train else 8)}
        if op == "add_norm":  # x, residual -> s, y; s, dy, ds -> dx, dresidual
            return {"bytes": n * e * (9 if train else 4), "flops": n * (24 if train else 10)}
        r = 1 if c["residual"] else 0  # the residual's gradient is dy itself
        return {"bytes": n * e * (2 + r + (2 if train else 0)), "flops": n * (4 if train else 2)}
    d = c["dim"]
    if op == "rotary":
        n = c["batch"] * c["tokens"] * d * (c["heads"] + c["kv_heads"])
        return {"bytes": n * e * (4 if train else 2) + c["batch"] * c["tokens"] * c["axes"] * 8, "flops": n * (6 if train else 3)}
    b, lq, l, h, kv, block = (c[n] for n in ("batch", "q_tokens", "tokens", "heads", "kv_heads", "block"))
    tq, tk = -(-lq // block), -(-l // block)
    nq, nk = b * lq * h * d, b * l * kv * d
    choose = {"bytes": (nq + nk) * e + b * kv * tq * c["top"] * 4, "flops": nq + nk + 2 * b * kv * tq * tk * d}
    if op == "select":
        return choose
    keys = min(c["top"] * block, l)
    read = min(nk, b * kv * tq * keys * d)  # key and value rows that are read at all
    a = {"bytes": (2 * nq + 2 * read) * e + b * kv * tq * c["top"] * 4, "flops": 4 * b * lq * h * d * keys}
    if train:  # q, k, v, o, do -> dq, dk, dv
        a = {"bytes": a["bytes"] + (4 * nq + 4 * nk) * e, "flops": a["flops"] * 3.5}
    if op == "serve":
        a = {"bytes": a["bytes"] + choose["bytes"], "flops": a["flops"] + choose["flops"]}
    return a


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------


def _exact_keep(n, p, seed, step, call):
    """Philox4x32-10 on unsigned 64-bit host arrays, the products' halves by unsigned arithmetic."""
    u = np.uint64
    low = u(0xFFFFFFFF)
    i = np.arange((n + 3) // 4, dtype=np.uint64)
    w0, w1 = i & low, i >> u(32)
    w2, w3 = np.full_like(i, u(call)), np.full_like(i, u(step & 0xFFFFFFFF))
    ka, kb = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for r in range(10):
        x, y = u(0xD2511F53) * w0, u(0xCD9E8D57) * w2
        w0, w1, w2, w3 = (y >> u(32)) ^ w1 ^ u(ka), y & low, (x >> u(32)) ^ w3 ^ u(kb), x & low
        ka, kb = (ka + 0x9E3779B9) % 2 ** 32, (kb + 0xBB67AE85) % 2 ** 32
    words = np.empty((i.size, 4), dtype=np.uint32)
    words[:, 0], words[:, 1], words[:, 2], words[:, 3] = w0, w1, w2, w3
    return words.reshape(-1)[:n] >= p * 2.0 ** 32


def _exact_rows(s, c):
    op = c["op"]
    x = s["x"].detach().double()
    n, m = x.shape
    out, z, drop = {}, x, None
    if op != "norm":
        seed, step = (int(v) for v in s["rng"].cpu())
        keep = torch.from_numpy(_exact_keep(n * m, c["p"], seed, step, 1 if op == "add_norm" else 2)).to(x.device).view(n, m)
        drop = keep.double() / (1.0 - c["p"])
        z = x * drop
        if "residual" in s:
            z = z + s["residual"].detach().double()
    if op == "dropout":
        dy = s["dy"].double() if c["train"] else None
        out["y"] = z
        if c["train"]:
            out["grads"] = [dy * drop] + ([dy] if c["residual"] else [])
        return out
    if op == "add_norm":
        out["s"] = z
    w, b = s["weight"].detach().double(), s["bias"].detach().double()
    var, mean = torch.var_mean(z, 1, correction=0)
    sd = torch.sqrt(var + 1e-5)
    hat = (z - mean[:, None]) / sd[:, None]
    out["y"] = torch.addcmul(b, hat, w)
    if c["train"]:
        dy = s["dy"].double()
        a = dy * w
        c1, c2 = a.sum(1) / m, torch.linalg.vecdot(a, hat) / m
        dz = (a - c1[:, None] - hat * c2[:, None]) / sd[:, None]
        dw, db = torch.linalg.vecdot(dy, hat, dim=0), dy.sum(0)
        if op == "norm":
            out["grads"] = [dz, dw, db]
        else:
            dz = dz + s["ds"].double()
            out["grads"] = [dz * drop, dz, dw, db]
    return out


def _exact_rotary(s, c):
    per = s["freqs"].numel() // c["axes"]
    pos = torch.stack([s["positions"][..., i // per] for i in range(s["freqs"].numel())], -1).double()
    turn = torch.polar(torch.ones_like(pos), pos * s["freqs"])[:, :, None]
    n = turn.shape[-1]

    def spin(x, z):
        x = x.detach().double()
        y = x.clone()
        even, odd = (slice(0, 2 * n, 2), slice(1, 2 * n, 2)) if c["interleaved"] else (slice(0, n), slice(n, 2 * n))
        u = torch.complex(x[..., even].contiguous(), x[..., odd].contiguous()) * z
        y[..., even], y[..., odd] = u.real, u.imag
        return y

    out = {"q": spin(s["q"], turn), "k": spin(s["k"], turn)}
    if c["train"]:
        out["grads"] = [spin(s["dq"], turn.conj()), spin(s["dk"], turn.conj())]
    return out


def _exact_choice(s, c):
    """Scene by scene, head by head: the means of the rows that count, and the places in descending order of (score, -place)."""
    b, kv, group, block = c["batch"], c["kv_heads"], c["heads"] // c["kv_heads"], c["block"]
    lq, l = c["q_tokens"], c["tokens"]
    tq, tk = -(-lq // block), -(-l // block)
    index = torch.full((b, kv, tq, c["top"]), -1, dtype=torch.int32, device=s["q"].device)
    for i in range(b):
        nq = lq if s["q_lengths"] is None else int(s["q_lengths"][i])
        nk = l if s["kv_lengths"] is None else int(s["kv_lengths"][i])
        if not nq or not nk:
            continue
        uq, uk = -(-nq // block), -(-nk // block)
        tile_q = torch.arange(nq, device=index.device) // block
        tile_k = torch.arange(nk, device=index.device) // block
        for j in range(kv):
            a = s["q"][i, :nq, j * group:(j + 1) * group].detach().double().mean(1)
            e = s["k"][i, :nk, j].detach().double()
            am = torch.zeros((uq, c["dim"]), dtype=torch.float64, device=a.device).index_add_(0, tile_q, a)
            em = torch.zeros((uk, c["dim"]), dtype=torch.float64, device=a.device).index_add_(0, tile_k, e)
            am, em = am / torch.bincount(tile_q)[:, None], em / torch.bincount(tile_k)[:, None]
            score = (am @ em.T).cpu().numpy()
            ok = np.ones((uq, uk), bool) if s["allowed"] is None else s["allowed"][:uq, :uk].cpu().numpy()
            order = np.argsort(np.where(ok, -score, np.inf), axis=1, kind="stable")[:, :c["top"]]
            got = np.where(np.take_along_axis(ok, order, 1), order, tk)
            got = np.sort(got, axis=1)
            index[i, j, :uq, :got.shape[1]] = torch.from_numpy(np.where(got == tk, -1, got)).to(index)
    return index


def _exact_attend(s, c, index):
    """Dense rows against all keys of the sequence, those outside the chosen blocks hidden, some tiles at a time."""
    b, lq, l, h, kv, d, block = (c[n] for n in ("batch", "q_tokens", "tokens", "heads", "kv_heads", "dim", "block"))
    dev, f8, scale = s["q"].device, torch.float64, c["dim"] ** -0.5
    train = c.get("train", False)
    o = torch.zeros((b, lq, h, d), dtype=f8, device=dev)
    dq, dk, dv = (torch.zeros((b, n, m, d), dtype=f8, device=dev) if train else None for n, m in ((lq, h), (l, kv), (l, kv)))
    tk = -(-l // block)
    some = max(1, min(4096, 400_000_000 // max(l, 1)) // block)
    for i in range(b):
        nq = lq if s["q_lengths"] is None else int(s["q_lengths"][i])
        nk = l if s["kv_lengths"] is None else int(s["kv_lengths"][i])
        for j in range(h):
            g = j // (h // kv)
            k, v = s["k"][i, :nk, g].detach().double(), s["v"][i, :nk, g].detach().double()
            for t0 in range(0, -(-nq // block), some):
                lo, hi = t0 * block, min(nq, (t0 + some) * block)
                at = index[i, g, t0:t0 + some].long()
                pick = torch.zeros((at.shape[0], tk + 1), dtype=torch.bool, device=dev)
                pick.scatter_(1, torch.where(at < 0, tk, at), True)
                hide = ~pick[:, :tk].repeat_interleave(block, 1)[:, :nk].repeat_interleave(block, 0)[:hi - lo]
                q = s["q"][i, lo:hi, j].detach().double()
                p = torch.softmax((q @ k.T * scale).masked_fill_(hide, -math.inf), 1)
                p = p.masked_fill_(hide, 0.0)  # rows that see nothing too
                o[i, lo:hi, j] = p @ v
                if train:
                    do = s["do"][i, lo:hi, j].double()
                    dv[i, :nk, g] += p.T @ do
                    e = p * (do @ v.T - torch.linalg.vecdot(do, o[i, lo:hi, j])[:, None]) * scale
                    dq[i, lo:hi, j] = e @ k
                    dk[i, :nk, g] += e.T @ q
    return {"o": o, "grads": [dq, dk, dv]} if train else {"o": o}


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        if case["op"] in ("norm", "add_norm", "dropout"):
            return _exact_rows(s, case)
        if case["op"] == "rotary":
            return _exact_rotary(s, case)
        if case["op"] == "attend":
            return _exact_attend(s, case, s["index"])
        index = _exact_choice(s, case)
        return {"index": index} if case["op"] == "select" else {"index": index, **_exact_attend(s, case, index)}
