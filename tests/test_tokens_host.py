"""View-token operators, what needs no GPU: the oracle's own checks (generator's known answer, gradients
against differences), the helpers' values, and every refusal of the public entry points and the C ABI."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import token_oracle as orc
from my_depthsplat_amd import _lib, tokens


def test_philox_known_answers():
    """The published known answers of philox4x32-10 (counter and key all 0, all ones)."""
    assert orc.philox4x32((0,) * 4, (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = 0xFFFFFFFF
    assert orc.philox4x32((ones,) * 4, (ones, ones)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    words = orc.philox4x32((3, 0, 7, 9), (5, 1))
    got = orc.philox4x32_arrays([orc.np.array([v], dtype=orc.np.uint64) for v in (3, 0, 7, 9)], (1 << 32) | 5)
    assert [int(g[0]) for g in got] == words


def directional(f, x, d, h=1e-5):
    return (f(x + h * d) - f(x - h * d)) / (2 * h)


def test_oracle_gradients_against_differences():
    g = torch.Generator().manual_seed(0)
    rnd = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    z, w, b, dy = rnd(5, 12), rnd(12), rnd(12), rnd(5, 12)
    y, xh, r, _ = orc.layer_norm(z, w, b, 1e-5)
    dz, dw, db = orc.layer_norm_grads(xh, r, dy, w)
    for i, (x, grad) in enumerate(((z, dz), (w, dw), (b, db))):
        d = rnd(*x.shape)
        args = [z, w, b]
        f = lambda v: float((orc.layer_norm(*(args[:i] + [v] + args[i + 1:]), 1e-5)[0] * dy).sum())  # noqa: B023,E731
        assert abs(directional(f, x, d) - float((grad * d).sum())) < 1e-6
    q, k, v, do = rnd(2, 70, 4, 8), rnd(2, 100, 2, 8), rnd(2, 100, 2, 8), rnd(2, 70, 4, 8)
    index = torch.tensor([[0, 2], [1, -1], [3, 2]], dtype=torch.int32).expand(2, 2, 3, 2)
    lens = dict(q_lengths=torch.tensor([70, 40]), kv_lengths=torch.tensor([100, 50]))
    out = orc.attention(q, k, v, index, 32, do=do, **lens)
    for i, name in enumerate(("dq", "dk", "dv")):
        args = [q, k, v]
        d = rnd(*args[i].shape)
        f = lambda x: float((orc.attention(*(args[:i] + [x] + args[i + 1:]), index, 32, **lens)["o"] * do).sum())  # noqa: B023,E731
        assert abs(directional(f, args[i], d) - float((out[name] * d).sum())) < 1e-5


def test_rotary_frequencies():
    f = tokens.rotary_frequencies(16, axes=2, device="cpu")
    assert f.dtype == torch.float64 and f.shape == (8,) and torch.equal(f[:4], f[4:])
    assert f[0] == 1.0 and abs(float(f[1]) - 10.0 ** -1) < 1e-15
    assert torch.allclose(tokens.rotary_frequencies(8, stretch=4.0, device="cpu"), tokens.rotary_frequencies(8, device="cpu") / 4)
    g, h = tokens.rotary_frequencies(64, stretch=8.0, trained=2048, device="cpu"), tokens.rotary_frequencies(64, device="cpu")
    turns = 2048 * h / (2 * math.pi)
    assert torch.allclose(g[turns >= 32], h[turns >= 32]) and torch.allclose(g[turns <= 1], h[turns <= 1] / 8)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and bool(((g < h) & (g > h / 8))[mid].all())
    for bad in (dict(part=6, axes=2), dict(part=0), dict(part=8, stretch=0.5), dict(part=8, base=0.0), dict(part=8, axes=0)):
        with pytest.raises(ValueError):
            tokens.rotary_frequencies(device="cpu", **bad)


def test_view_positions():
    p = tokens.view_positions(2, 3, 5, device="cpu")
    assert p.shape == (30, 2) and p[7].tolist() == [1, 2] and torch.equal(p[:15], p[15:])


x = torch.zeros(4, 6)
w = torch.ones(6)
rng = torch.zeros(2, dtype=torch.int64)
half = torch.float16


@pytest.mark.parametrize("call", [
    lambda: tokens.layer_norm(x.double()),
    lambda: tokens.layer_norm(torch.zeros(())),
    lambda: tokens.layer_norm(torch.zeros(4, 0)),
    lambda: tokens.layer_norm(x, w[:5]),
    lambda: tokens.layer_norm(x, w.to(half)),
    lambda: tokens.layer_norm(x.to(half), w, w.to(half)),
    lambda: tokens.layer_norm(x, w, w, eps=-1.0),
    lambda: tokens.layer_norm(x, w, w, eps=float("nan")),
    lambda: tokens.dropout(x, -0.1, rng),
    lambda: tokens.dropout(x, 1.5, rng),
    lambda: tokens.dropout(x, float("nan"), rng),
    lambda: tokens.dropout(x, 0.5),
    lambda: tokens.dropout(x, 0.5, rng.int()),
    lambda: tokens.dropout(x, 0.5, rng[:1]),
    lambda: tokens.dropout(x, 0.5, torch.zeros(4, dtype=torch.int64)[::2]),
    lambda: tokens.dropout(x, 0.5, rng, call=-1),
    lambda: tokens.dropout(x, 0.5, rng, call=1 << 32),
    lambda: tokens.dropout(x.long(), 0.5, rng),
    lambda: tokens.dropout(x, 0.5, rng, residual=x[:3]),
    lambda: tokens.dropout(x, 0.5, rng, residual=x.to(half)),
    lambda: tokens.dropout_add_layer_norm(x, x[:, :5], w, w),
    lambda: tokens.dropout_add_layer_norm(x, x.to(half), w, w),
    lambda: tokens.dropout_add_layer_norm(x, x, w, w, p=0.5),
    lambda: tokens.layer_norm(x[:1, :1].expand(1, (1 << 32) + 16)),
    lambda: tokens.layer_norm(x[:1, :2].expand(1 << 31, 2)),
])
def test_row_refusals(call):
    with pytest.raises(ValueError):
        call()


q4, k4 = torch.zeros(2, 5, 4, 16), torch.zeros(2, 5, 2, 16)
pos, fr = torch.zeros(5, dtype=torch.int64), torch.ones(4, dtype=torch.float64)


@pytest.mark.parametrize("call", [
    lambda: tokens.rotary(q4[0], None, pos, fr),
    lambda: tokens.rotary(q4, k4[:1], pos, fr),
    lambda: tokens.rotary(q4, k4[..., :8], pos, fr),
    lambda: tokens.rotary(q4, k4.to(half), pos, fr),
    lambda: tokens.rotary(q4.double(), None, pos, fr),
    lambda: tokens.rotary(q4, k4, pos[:4], fr),
    lambda: tokens.rotary(q4, k4, torch.zeros(3, 5, 1), fr),
    lambda: tokens.rotary(q4, k4, pos.double(), fr),
    lambda: tokens.rotary(q4, k4, pos, fr.float()),
    lambda: tokens.rotary(q4, k4, pos, torch.ones(9, dtype=torch.float64)),
    lambda: tokens.rotary(q4, k4, torch.zeros(5, 3, dtype=torch.int64), fr),
    lambda: tokens.rotary(q4, k4, torch.zeros(5, 0, dtype=torch.int64), fr),
    lambda: tokens.rotary(q4, k4, pos.float().requires_grad_(True), fr),
    lambda: tokens.rotary(q4, k4, pos, fr.clone().requires_grad_(True)),
    lambda: tokens.rotary(q4[:, :, :1].expand(2, 5, 65536, 16), None, pos, fr),
    lambda: tokens.rotary(q4, k4[:, :, :1].expand(2, 5, (1 << 32) + 2, 16), pos, fr),
])
def test_rotary_refusals(call):
    with pytest.raises(ValueError):
        call()


idx = torch.zeros(2, 2, 1, 3, dtype=torch.int32)


@pytest.mark.parametrize("call", [
    lambda: tokens.select_blocks(q4, k4, 2, block=16),
    lambda: tokens.select_blocks(q4, k4, 0),
    lambda: tokens.select_blocks(q4[:, :, :3], k4, 2),
    lambda: tokens.select_blocks(q4[:, :, :1].expand(2, 5, (1 << 32) + 2, 16), k4, 2),
    lambda: tokens.select_blocks(q4, k4[:, :1].expand(2, 1 << 31, 2, 16), 2),
    lambda: tokens.select_blocks(q4, k4[:, :, :0], 2),
    lambda: tokens.select_blocks(q4, k4.to(half), 2),
    lambda: tokens.select_blocks(torch.zeros(1, 2, 1, 257), torch.zeros(1, 2, 1, 257), 2),
    lambda: tokens.select_blocks(q4, k4, 2, q_lengths=torch.zeros(3, dtype=torch.int32)),
    lambda: tokens.select_blocks(q4, k4, 2, kv_lengths=torch.zeros(2)),
    lambda: tokens.select_blocks(q4, k4, 2, allowed=torch.zeros(1, 1)),
    lambda: tokens.select_blocks(q4, k4, 2, allowed=torch.zeros(2, 1, dtype=torch.bool)),
    lambda: tokens.block_sparse_attention(q4, k4, k4[:, :4], idx),
    lambda: tokens.block_sparse_attention(q4, k4, k4.to(half), idx),
    lambda: tokens.block_sparse_attention(q4, k4, k4, idx.long()),
    lambda: tokens.block_sparse_attention(q4, k4, k4, idx[:, :1]),
    lambda: tokens.block_sparse_attention(q4, k4, k4, idx[..., :0]),
    lambda: tokens.block_sparse_attention(q4, k4, k4, idx.expand(2, 2, 1, 3).repeat(1, 1, 1, 342)),
    lambda: tokens.block_sparse_attention(q4[..., :12], k4[..., :12], k4[..., :12], idx),
    lambda: tokens.block_sparse_attention(q4.repeat(1, 1, 1, 9), k4.repeat(1, 1, 1, 9), k4.repeat(1, 1, 1, 9), idx),
    lambda: tokens.block_sparse_attention(torch.zeros(1, 2, 1025, 8), torch.zeros(1, 2, 1, 8), torch.zeros(1, 2, 1, 8), idx[:1, :1]),
    lambda: tokens.block_sparse_attention(q4, k4, k4, idx, block=48),
    lambda: tokens.block_sparse_attention(q4, k4, k4, idx, kv_lengths=torch.zeros(1, 2, dtype=torch.int32)),
])
def test_attention_refusals(call):
    with pytest.raises(ValueError):
        call()


@pytest.mark.skipif(torch.cuda.is_available(), reason="GPU present")
@pytest.mark.parametrize("call", [
    lambda: tokens.layer_norm(x, w, w),
    lambda: tokens.dropout(x, 0.5, rng),
    lambda: tokens.dropout_add_layer_norm(x, x, w, w),
    lambda: tokens.rotary(q4, k4, pos, fr),
    lambda: tokens.select_blocks(q4, k4, 2),
    lambda: tokens.block_sparse_attention(q4, k4, k4, idx),
])
def test_cpu_tensors_fail_loudly(call):
    if not _lib.LIB_PATH.exists():
        pytest.skip("extension not built")
    with pytest.raises(_lib.DsplatError):
        call()


def test_abi_refusals():
    """Sizes, types and missing pointers are refused before any HIP call."""
    if not _lib.LIB_PATH.exists():
        pytest.skip("extension not built")
    lib = _lib.load()
    buf = ctypes.create_string_buffer(4096)
    s3 = (ctypes.c_int64 * 3)(1, 1, 1)

    def refused(rc, text):
        assert rc == 1 and text in lib.dsplat_last_error(), lib.dsplat_last_error()

    refused(lib.dtk_dropout(-1, 0, buf, None, 0.5, buf, 0, buf, None), b"bad sizes")
    refused(lib.dtk_dropout(4, 3, buf, None, 0.5, buf, 0, buf, None), b"bad type")
    refused(lib.dtk_dropout(4, 0, buf, None, 1.5, buf, 0, buf, None), b"p must be")
    refused(lib.dtk_dropout(4, 0, buf, None, 0.5, None, 0, buf, None), b"null pointer")
    assert lib.dtk_dropout(0, 0, None, None, 0.5, None, 0, None, None) == 0
    refused(lib.dtk_layer_norm_fwd(4, 0, 0, 0, buf, None, None, None, 1e-5, 0.0, None, 0, None, buf, None, None, None), b"bad sizes")
    refused(lib.dtk_layer_norm_fwd(4, 8, 0, 1, buf, None, None, None, 1e-5, 0.0, None, 0, None, buf, None, None, None), b"bad types")
    refused(lib.dtk_layer_norm_fwd(4, 8, 0, 0, buf, None, None, None, 1e-5, 0.5, None, 0, None, buf, None, None, None), b"dropout needs")
    refused(lib.dtk_layer_norm_fwd(4, 8, 0, 0, buf, buf, None, None, 1e-5, 0.0, None, 0, None, buf, None, None, None), b"null pointer")
    refused(lib.dtk_layer_norm_bwd(4, 8, 0, 0, buf, buf, buf, None, buf, buf, 0, 0.0, None, 0, buf, None, None, None, None, None), b"without a residual")
    refused(lib.dtk_layer_norm_bwd(4, 8, 0, 0, buf, buf, None, None, buf, buf, 0, 0.0, None, 0, buf, None, buf, None, None, None), b"null pointer")
    rot = lambda D, F, axes, dt, pt, q: lib.dtk_rotary(1, 2, 1, 0, D, F, axes, 0, 0, dt, pt, q, s3, None, None, buf, s3, buf, 1.0, buf, None, None)  # noqa: E731
    refused(rot(0, 0, 1, 0, 4, buf), b"bad sizes")
    refused(rot(8, 5, 1, 0, 4, buf), b"bad number")
    refused(rot(8, 3, 2, 0, 4, buf), b"bad number")
    refused(rot(8, 4, 1, 3, 4, buf), b"bad types")
    refused(rot(8, 4, 1, 0, 4, None), b"null pointer")
    sel = lambda Hq, Hkv, D, block, top: lib.dtk_select_blocks(1, 9, 9, Hq, Hkv, D, block, top, 0, buf, s3, buf, s3, None, None, None, buf, None, None)  # noqa: E731
    refused(sel(3, 2, 8, 64, 2), b"bad sizes")
    refused(sel(2, 2, 8, 48, 2), b"block must be")
    refused(sel(2, 2, 8, 64, 2), b"null pointer")
    at = lambda **kw: _lib.Attention(**{**dict(Lq=9, Lk=9, B=1, Hq=2, Hkv=1, D=8, block=64, top=2, dtype=0, scale=1.0), **kw})  # noqa: E731
    for kw, text in ((dict(Hq=3, Hkv=2), b"bad sizes"), (dict(top=1025), b"bad sizes"), (dict(D=12), b"multiple of 8"),
                     (dict(D=136), b"multiple of 8"), (dict(block=16), b"block must be"), (dict(dtype=4), b"bad type"),
                     (dict(Hq=1025), b"more than 1024"), (dict(k_strides=(0, 1 << 24, 8)), b"token stride"),
                     (dict(v_strides=(0, -8, 8)), b"token stride"), (dict(), b"null pointer")):
        refused(lib.dtk_block_sparse_attention_fwd(ctypes.byref(at(**kw)), None, None), text)
        refused(lib.dtk_block_sparse_attention_bwd(ctypes.byref(at(**kw)), None, None, None, None, None, None, None), text)
    refused(lib.dtk_block_sparse_attention_fwd(None, None, None), b"null pointer")
