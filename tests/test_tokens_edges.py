"""View-token operators and their layer at the edges of what they allow."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import token_oracle as orc
from my_depthsplat_amd import _lib, tokens
from test_tokens_gpu import check_attention

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


# ---- f16: gradients of very different sizes ------------------------------------------------


def f16_gradients(q, k, v, do, see, scale):
    """64-bit inputs of one head each, q, do [L, D], k, v [Lk, D], see [L, Lk] -> name -> (gradient, bound). Each row's
    terms are counted by its own |do|: p and ds are rounded to f16 for their products, half a step of their value or, far
    below the largest of their column, of f16's smallest numbers relative to it: the column's largest is
    taken to 2^12 at least, so 2^-25 / 2^12 of it; p is at most 1 and taken times 2^12."""
    h = orc.half_step(F16)
    x = (q @ k.T * scale).masked_fill(~see, -math.inf)
    p = torch.softmax(x, -1)
    o, dp = p @ v, do @ v.T
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    noise = (2 * q.shape[1] + int(see.sum(-1).max()) + 32) * orc.E32 * (1 + float((q.abs() @ k.abs().T).max()) * abs(scale))
    # delta is of o as it was rounded
    e = h * ds.abs() + p * (h * (do.abs() * o.abs()).sum(-1, keepdim=True)
                            + noise * (do.abs() @ v.abs().T + (do.abs() * (p @ v.abs())).sum(-1, keepdim=True)))
    low = 2.0 ** -37
    eq, ek = (e + see * low * ds.abs().amax(1, keepdim=True)), (e + see * low * ds.abs().amax(0, keepdim=True))
    ep = (h + noise) * p + see * low
    rows = q.shape[0] * orc.E32
    out = {"dq": (ds @ k * scale, eq @ k.abs() * abs(scale)),
           "dk": (ds.T @ q * scale, (ek + rows * ds.abs()).T @ q.abs() * abs(scale)),
           "dv": (p.T @ do, (ep + rows * p).T @ do.abs())}
    return {n: (g, b + h * g.abs() + orc.tiny(F16)) for n, (g, b) in out.items()}


def check_f16_gradients(gpu, q, k, v, do, index, block, scale, only=("dq", "dk", "dv")):
    """[B, L, D] f16 host tensors of one head"""
    leaves = [x[:, :, None].to(gpu).requires_grad_(True) for x in (q, k, v)]
    o = tokens.block_sparse_attention(*leaves, index.to(gpu), block=block, scale=scale)
    got = torch.autograd.grad(o, leaves, do[:, :, None].to(gpu))
    for b in range(q.shape[0]):
        see = torch.zeros(q.shape[1], k.shape[1], dtype=torch.bool)
        for tile in range(index.shape[2]):
            for j in index[b, 0, tile].tolist():
                if j >= 0:
                    see[tile * block:(tile + 1) * block, j * block:(j + 1) * block] = True
        want = f16_gradients(*(x[b].double() for x in (q, k, v, do)), see, scale)
        for name, g in zip(("dq", "dk", "dv"), got):
            if name in only:
                orc.assert_within(g[b, :, 0], *want[name], f"{name} of scene {b}")


def f16(*shape, seed=0, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(F16)


@gpu_only
@pytest.mark.parametrize("D,block", [(32, 32), (64, 64), (96, 128), (128, 64)])
def test_f16_gradients_of_a_scene_do_not_depend_on_anothers(gpu, D, block):
    """Scenes whose do are 2^8, 1 and 2^-8: each within its own roundings, and the bits of the scene by itself."""
    L = 4 * block
    q, k, v, do = (f16(3, L, D, seed=i) for i in range(4))
    do = do * torch.tensor([2.0 ** 8, 1.0, 2.0 ** -8]).to(F16)[:, None, None]
    # (few of f16's smallest numbers in do itself: those stay as they are)
    index = torch.arange(4, dtype=torch.int32).expand(3, 1, 4, 4).contiguous()
    check_f16_gradients(gpu, q, k, v, do, index, block, D ** -0.5)
    together = [x[:, :, None].to(gpu).requires_grad_(True) for x in (q, k, v)]
    gd = do[:, :, None].to(gpu)
    all_of = torch.autograd.grad(tokens.block_sparse_attention(*together, index.to(gpu), block=block), together, gd)
    for b in range(3):
        alone = [x[b:b + 1].detach().requires_grad_(True) for x in together]
        one = torch.autograd.grad(tokens.block_sparse_attention(*alone, index[b:b + 1].to(gpu), block=block), alone, gd[b:b + 1])
        assert all(torch.equal(x[b:b + 1], y) for x, y in zip(all_of, one)), b


@gpu_only
@pytest.mark.parametrize("block,Lq,G", [(32, 128, 1), (64, 256, 1), (128, 256, 1), (64, 1, 1)])
def test_f16_gradients_of_a_row_do_not_depend_on_its_neighbours(gpu, block, Lq, G):
    """Every other row has a do of 2^10 and zeros in the second half of q's channels, so dk's second half comes from the rows between
    alone, whose do is 2^-4; the large rows come first in some units and last in others."""
    D, L = 64, Lq
    q, k, v, do = f16(1, L, D, seed=1), f16(1, 3 * block, D, seed=2), f16(1, 3 * block, D, seed=3), f16(1, L, D, seed=4)
    large = torch.zeros(L, dtype=torch.bool)
    large[::2] = True
    large[32:64] = False
    large[64:96] = True
    q[:, large, D // 2:] = 0
    do = torch.where(large[:, None], do * 2.0 ** 10, do * 2.0 ** -4).to(F16)
    index = torch.arange(3, dtype=torch.int32).expand(1, 1, -(-L // block), 3).contiguous()
    check_f16_gradients(gpu, q, k, v, do, index, block, D ** -0.5)


@gpu_only
@pytest.mark.parametrize("block", [32, 64, 128])
def test_f16_gradients_of_unlikely_keys(gpu, block):
    """The second block's keys get a share of 2^-17 each: below f16's normal numbers, yet their gradients, of a do of 2^10, are not."""
    D, L = 32, 2 * block
    q, k, v, do = f16(1, L, D, seed=1, scale=0.3), f16(1, L, D, seed=2, scale=0.3), f16(1, L, D, seed=3), f16(1, L, D, seed=4, scale=2.0 ** 10)
    q[..., 0], k[:, :block, 0], k[:, block:, 0] = 1.0, 0.0, -(17 - math.log2(block)) * math.log(2)
    index = torch.arange(2, dtype=torch.int32).expand(1, 1, 2, 2).contiguous()
    check_f16_gradients(gpu, q, k, v, do, index, block, 1.0)


@gpu_only
def test_f16_gradients_of_infinite_and_zero_rows(gpu):
    """Rows whose do is 0 give 0; one of infinity in one scene leaves the others' gradients as they are."""
    q, k, v, do = (f16(2, 128, 1, 64, seed=i).to(gpu) for i in range(4))
    index = torch.arange(2, device=gpu, dtype=torch.int32).expand(2, 1, 2, 2).contiguous()

    def grads(g):
        leaves = [x.detach().requires_grad_(True) for x in (q, k, v)]
        return torch.autograd.grad(tokens.block_sparse_attention(*leaves, index), leaves, g)

    want = grads(do)
    bad = do.clone()
    bad[0, 5, 0, 3] = math.inf
    got = grads(bad)
    assert all(torch.equal(a[1], b[1]) for a, b in zip(got, want))
    keep = [i for i in range(128) if i != 5]
    assert torch.equal(got[0][0, keep], want[0][0, keep]) and not got[0][0, 5].isfinite().all()
    assert all(not x.any() for x in grads(torch.zeros_like(do)))


# ---- the head and its layer -----------------------------------------------------------------


def small_head(**kw):
    from my_depthsplat_amd.training import GaussianHead
    torch.manual_seed(0)
    return GaussianHead(10, **{**dict(width=24, down=2, token_layers=2, token_heads=2, token_top=2, seed=7), **kw})


def scene(gpu, t=F32):
    torch.manual_seed(1)
    return torch.rand(2, 3, 3, 24, 16, device=gpu).to(t), torch.rand(2, 3, 24 * 16, 1, 1, device=gpu).to(t)


@pytest.mark.parametrize("cast", [lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.float(), lambda m: m.double().float(),
                                  lambda m: m.to(BF16), lambda m: m.to("meta").to_empty(device="cpu")])
def test_head_frequencies_keep_64_bits_through_casts(cast):
    want = small_head().freqs.clone()
    head = cast(small_head())
    assert head.freqs.dtype == torch.float64 and torch.equal(head.freqs, want)
    assert head.rng.dtype == torch.int64 and "freqs" not in head.state_dict()
    kept = head.freqs
    assert head.float().freqs is kept and head.cpu().freqs is kept  # (a captured graph may hold it)
    assert small_head(token_layers=0).bfloat16().layers is None


@gpu_only
@pytest.mark.parametrize("t", TYPES)
def test_head_in_each_type_trains(gpu, t):
    """A module cast: every parameter gets a finite gradient, and the output is within a tenth of the f32 head's norm (some 20
    roundings of 2^-8 in turn)."""
    head = small_head(token_dropout=0.1)
    want = small_head(token_dropout=0.1).to(gpu)(*scene(gpu)).detach()
    head = head.to(gpu).to(t)
    y = head(*scene(gpu, t))
    assert float((y.detach().float() - want).norm() / want.norm()) < 0.1
    y.float().square().sum().backward()
    for n, p in head.named_parameters():
        assert p.grad is not None and p.grad.dtype == t and bool(p.grad.isfinite().all()) and bool((p.grad != 0).any()), n


@gpu_only
@pytest.mark.parametrize("t", [BF16, F16])
def test_head_and_layer_under_autocast(gpu, t):
    """The products in 16 bits, the sum of the layers in the rows' own type: within a tenth of the result without (some 20 roundings
    of 2^-8 in turn), finite gradients in the parameters' type; the layer by itself keeps its input's type."""
    head = small_head(token_dropout=0.1).to(gpu)
    want = small_head(token_dropout=0.1).to(gpu)(*scene(gpu)).detach()
    with torch.autocast("cuda", t):
        y = head(*scene(gpu))
    assert float((y.detach().float() - want).norm() / want.norm()) < 0.1
    y.float().square().sum().backward()
    for n, p in head.named_parameters():
        assert p.grad is not None and p.grad.dtype == F32 and bool(p.grad.isfinite().all()), n
    layer, freqs = head.layers[0].eval(), head.freqs
    pos = tokens.view_positions(2, 5, 6, gpu)
    x = torch.randn(2, 60, 48, device=gpu, requires_grad=True)
    plain = layer(x, pos, freqs).detach()
    with torch.autocast("cuda", t):
        z = layer(x, pos, freqs)
    assert z.dtype == F32 and float((z.detach() - plain).norm() / plain.norm()) < 0.05
    (g,) = torch.autograd.grad(z.square().sum(), x)
    assert g.dtype == F32 and bool(g.isfinite().all())


@gpu_only
@pytest.mark.parametrize("reentrant", [False, True])
def test_head_under_activation_checkpointing(gpu, reentrant):
    """A forward that is computed again draws the same masks if its generator state is an argument: the gradients of the call
    without, in several steps at once; without that argument it is an error, not another step's masks."""
    from torch.utils.checkpoint import checkpoint
    images, depths = scene(gpu)
    images.requires_grad_(True)  # (a reentrant checkpoint needs an input that asks for a gradient)
    head = small_head(token_dropout=0.3).to(gpu)

    def grads(run):
        head.zero_grad()
        head.rng.copy_(torch.tensor([7, 0]))
        outs = [run(head.next_rng()) for _ in range(2)]
        assert head.rng.tolist() == [7, 2]
        sum((y * y).sum() for y in outs).backward()
        assert head.rng.tolist() == [7, 2]
        return [y.detach() for y in outs], [p.grad.clone() for p in head.parameters()]

    want, want_grads = grads(lambda rng: head(images, depths, rng))
    got, got_grads = grads(lambda rng: checkpoint(head, images, depths, rng, use_reentrant=reentrant))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    # (torch's convolutions' weight gradients may add in any order)
    assert all(float((a - b).norm()) <= 1e-5 * float(b.norm()) for a, b in zip(got_grads, want_grads))
    y = checkpoint(head, images, depths, use_reentrant=reentrant)
    with pytest.raises(RuntimeError, match="next_rng"):
        y.sum().backward()
    with torch.no_grad():
        head.rng.copy_(torch.tensor([7, 0]))
        assert torch.equal(head(images, depths), want[0]) and head.rng.tolist() == [7, 1]
    dry = small_head(token_dropout=0.0).to(gpu)  # nothing is drawn, so nothing can differ
    checkpoint(dry, images, depths, use_reentrant=reentrant).sum().backward()
    assert dry.rng.tolist() == [7, 1]


# ---- calls that are refused -----------------------------------------------------------------


def dual_calls():
    x, w = torch.randn(4, 8), torch.ones(8)
    q, k = torch.randn(2, 5, 4, 16), torch.randn(2, 5, 2, 16)
    rng, index = torch.zeros(2, dtype=torch.int64), torch.zeros(2, 2, 1, 1, dtype=torch.int32)
    pos, freqs = torch.zeros(5), torch.ones(4, dtype=torch.float64)
    T = tokens
    return [((x,), lambda a: T.layer_norm(a)), ((w,), lambda a: T.layer_norm(x, a)), ((w,), lambda a: T.layer_norm(x, w, a)),
            ((x,), lambda a: T.dropout(a, 0.5, rng)), ((x,), lambda a: T.dropout(x, 0.0, residual=a)),
            ((x,), lambda a: T.dropout_add_layer_norm(a, x)), ((x,), lambda a: T.dropout_add_layer_norm(x, a)),
            ((w,), lambda a: T.dropout_add_layer_norm(x, x, a)), ((w,), lambda a: T.dropout_add_layer_norm(x, x, w, a)),
            ((q,), lambda a: T.rotary(a, k, pos, freqs)), ((k,), lambda a: T.rotary(q, a, pos, freqs)),
            ((pos,), lambda a: T.rotary(q, k, a, freqs)), ((freqs,), lambda a: T.rotary(q, k, pos, a)),
            ((q,), lambda a: T.block_sparse_attention(a, k, k, index)), ((k,), lambda a: T.block_sparse_attention(q, a, k, index)),
            ((k,), lambda a: T.block_sparse_attention(q, k, a, index))]


@pytest.mark.parametrize("case", range(16))
def test_forward_mode_derivatives_are_refused(case):
    """A tangent that the result would lose is an error, not a derivative of 0; outside its level nothing is refused for it."""
    import torch.autograd.forward_ad as fw
    if not _lib.LIB_PATH.exists():
        pytest.skip("extension not built")
    (t,), call = dual_calls()[case]
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(fw.make_dual(t, torch.ones_like(t)))
    with pytest.raises(_lib.DsplatError):  # a CPU tensor
        call(t)


@gpu_only
def test_forward_mode_derivatives_where_nothing_is_done(gpu):
    """p = 0 returns x with its tangent; a tangent taken off is no obstacle."""
    import torch.autograd.forward_ad as fw
    x = torch.randn(4, 8, device=gpu)
    with fw.dual_level():
        d = fw.make_dual(x, torch.ones_like(x))
        assert tokens.dropout(d, 0.0) is d
        assert torch.equal(tokens.layer_norm(fw.unpack_dual(d).primal), tokens.layer_norm(x))


@pytest.mark.parametrize("scale", [math.nan, math.inf, -math.inf])
def test_attention_scale_that_is_no_number_is_refused(scale):
    if not _lib.LIB_PATH.exists():
        pytest.skip("extension not built")
    q, index = torch.zeros(1, 5, 1, 8), torch.zeros(1, 1, 1, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="scale"):
        tokens.block_sparse_attention(q, q, q, index, scale=scale)
    a = _lib.Attention(Lq=9, Lk=9, B=1, Hq=2, Hkv=1, D=8, block=64, top=2, dtype=0, scale=scale)
    assert _lib.load().dtk_block_sparse_attention_fwd(ctypes.byref(a), None, None) == 1
    assert b"scale" in _lib.load().dsplat_last_error()


def test_abi_sizes_that_do_not_fit_end_no_process():
    """Workspace sizes of arguments that the call itself refuses are 0 (no division by 0); 2 F past 32 bits is refused."""
    if not _lib.LIB_PATH.exists():
        pytest.skip("extension not built")
    lib = _lib.load()
    at = lambda **kw: _lib.Attention(**{**dict(Lq=900, Lk=900, B=1, Hq=2, Hkv=1, D=8, block=64, top=2, dtype=0, scale=1.0), **kw})  # noqa: E731
    sizes = (lib.dtk_block_sparse_attention_fwd_workspace_size, lib.dtk_block_sparse_attention_bwd_workspace_size)
    assert sizes[1](ctypes.byref(at())) > 0
    for kw in (dict(Hq=1, Hkv=2), dict(Hq=3, Hkv=2), dict(block=256), dict(block=48), dict(block=1 << 30), dict(D=0), dict(D=4096),
               dict(top=0), dict(top=-5), dict(top=2000), dict(Hq=2000), dict(Lq=1 << 40), dict(Lk=1 << 40), dict(B=1 << 20),
               dict(B=-1), dict(dtype=7)):
        for size in sizes:
            assert size(ctypes.byref(at(**kw))) == 0, kw
    assert all(size(None) == 0 for size in sizes)
    buf, s3 = ctypes.create_string_buffer(4096), (ctypes.c_int64 * 3)(1, 1, 1)
    for F in (1 << 30, (1 << 30) + 4, 0x7FFFFFFF):
        rc = lib.dtk_rotary(1, 2, 1, 0, 8, F, 1, 0, 0, 0, 4, buf, s3, None, None, buf, s3, buf, 1.0, buf, None, None)
        assert rc == 1 and b"bad number" in lib.dsplat_last_error(), F
    assert lib.dtk_select_blocks_workspace_size(1, 1 << 40, 9, 1, 8, 64) == 0
    assert lib.dtk_select_blocks_workspace_size(1, 9, 9, 1, 8, 48) == 0


@gpu_only
@pytest.mark.parametrize("long,short", [(2 ** 32, 300), (2 ** 40 + 7, 300), (2 ** 31, 300), (-2 ** 32 + 50, 0), (-2 ** 31 - 1, 0)])
def test_64_bit_lengths_past_32_bits(gpu, long, short):
    """Lengths are counted as they are: one behind the sequence's end means all of it, a negative one nothing."""
    q, k = torch.randn(1, 300, 1, 16, device=gpu), torch.randn(1, 300, 1, 16, device=gpu)
    far, near = (dict(q_lengths=torch.tensor([n], device=gpu), kv_lengths=torch.tensor([n], device=gpu)) for n in (long, short))
    index = tokens.select_blocks(q, k, 3, block=32, **near)
    assert torch.equal(tokens.select_blocks(q, k, 3, block=32, **far), index)
    index = tokens.select_blocks(q, k, 3, block=32)
    assert torch.equal(tokens.block_sparse_attention(q, k, k, index, block=32, **far),
                       tokens.block_sparse_attention(q, k, k, index, block=32, **near))


# ---- the choice of blocks -------------------------------------------------------------------


@gpu_only
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("blocks", [3, 200, 700, 2100])
@pytest.mark.parametrize("block,rows,value", [(128, 75, 1.75), (128, 91, 1.5), (64, 49, -1.0), (32, 13, 1.375), (128, 127, -1.25)])
def test_a_shorter_last_block_ties_with_the_others(gpu, t, blocks, block, rows, value):
    """Rows all equal: every block's mean is that value (a mean by a rounded reciprocal is not), so the lowest are chosen, of
    either sign."""
    k = torch.zeros(1, (blocks - 1) * block + rows, 1, 8, device=gpu, dtype=t)
    k[..., 0] = value
    q = torch.zeros(1, block + rows, 1, 8, device=gpu, dtype=t)
    q[..., 0] = 1.0
    for sign in (1, -1):
        assert tokens.select_blocks(q * sign, k, 2, block=block).flatten().tolist() == [0, 1] * 2


# ---- layer norm -----------------------------------------------------------------------------


@gpu_only
@pytest.mark.parametrize("add", [False, True])
@pytest.mark.parametrize("width", [8, 64, 512, 2048, 8192])
def test_layer_norm_gradients_beside_a_large_mean(gpu, add, width):
    """Rows of 1234568 and 1234560 in turn: every sum that the mean takes is exact in 32 bits (4 times whole numbers below 2^24, or
    such times a power of two), so the backward has no more to lose than its own roundings of numbers near 1 (64 of them in a
    chain at most; the weights' over 9 rows). (The mean times 1 / deviation, about 308641, rounded and subtracted: 2^-6.)"""
    g = torch.Generator().manual_seed(width)
    x = torch.tensor([1234568.0, 1234560.0]).repeat(9, width // 2)
    w, dy = torch.randn(width, generator=g), torch.randn(9, width, generator=g)
    leaves = [v.to(gpu).requires_grad_(True) for v in (x, w)]
    y = (tokens.dropout_add_layer_norm(leaves[0], torch.zeros_like(leaves[0]), leaves[1])[1] if add
         else tokens.layer_norm(leaves[0], leaves[1]))
    got = torch.autograd.grad(y, leaves, dy.to(gpu))
    _, xh, r, _ = orc.layer_norm(x.double(), w.double(), None, 1e-5)
    dz, dw, _ = orc.layer_norm_grads(xh, r, dy.double(), w.double())
    a = (dy * w).double().abs()
    orc.assert_within(got[0], dz, 64 * orc.E32 * (a + 2 * a.mean(-1, keepdim=True)), "dx")
    orc.assert_within(got[1], dw, 64 * orc.E32 * dy.double().abs().sum(0), "dw")


@gpu_only
@pytest.mark.parametrize("t", TYPES)
def test_attention_gradients_that_nobody_asks_for_are_not_taken(gpu, t):
    """Each subset's gradients are those of all three, to the bit; with frozen keys and values no memory is taken for theirs."""
    q, do = (torch.randn(1, 64, 2, 64, device=gpu).to(t) for _ in range(2))
    k, v = (torch.randn(1, 1 << 16, 1, 64, device=gpu).to(t) for _ in range(2))
    index = torch.tensor([[[[3, 700, 1023, 5]]]], dtype=torch.int32, device=gpu)

    def grads(asked):
        leaves = [x.detach().requires_grad_(n in asked) for n, x in zip("qkv", (q, k, v))]
        o = tokens.block_sparse_attention(*leaves, index)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        o.backward(do)
        torch.cuda.synchronize()
        return [x.grad for x in leaves], torch.cuda.max_memory_allocated() - held

    want, _ = grads("qkv")
    for asked in ("q", "k", "v", "qk", "qv", "kv"):
        got, more = grads(asked)
        assert all((a is None) == (n not in asked) and (a is None or torch.equal(a, b)) for n, a, b in zip("qkv", got, want)), asked
        if asked == "q":
            assert more < k.numel() * k.element_size(), more
    qr, kr = (torch.randn(1, 5, 2, 16, device=gpu) for _ in range(2))
    pos, freqs = torch.arange(5, device=gpu), tokens.rotary_frequencies(16, device=gpu)
    both = [x.clone().requires_grad_(True) for x in (qr, kr)]
    want = torch.autograd.grad(sum(x.sum() for x in tokens.rotary(*both, pos, freqs)), both)
    for i in range(2):
        one = [x.clone().requires_grad_(j == i) for j, x in enumerate((qr, kr))]
        (got,) = torch.autograd.grad(sum(x.sum() for x in tokens.rotary(*one, pos, freqs)), one[i])
        assert torch.equal(got, want[i])


# ---- the largest groups of heads and lists, a first call that is captured, a cache that sequences share ---------------


@gpu_only
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("block,Lq,D", [(32, 3, 8), (64, 1, 128), (128, 33, 24)])
def test_attention_of_1024_heads_to_one(gpu, t, block, Lq, D):
    check_attention(gpu, t, 1, Lq, 2 * block - 5, 1024, 1, D, block, 3, seed=block)


@gpu_only
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("Lq,D,Hq", [(1, 128, 1), (40, 128, 1), (64, 32, 2), (130, 128, 1)])
def test_attention_of_lists_of_1024(gpu, t, Lq, D, Hq):
    check_attention(gpu, t, 1, Lq, 1030 * 32 - 9, Hq, 1, D, 32, 1024, seed=Lq)


@gpu_only
@pytest.mark.parametrize("t", [F32, F16])
def test_attention_captured_without_a_call_before(gpu, t):
    """Kernels of more LDS than they get unasked, whose first launch is the captured one."""
    q, k, v, do = (torch.randn(2, 300, h, 104, device=gpu).to(t).requires_grad_(i < 3) for i, h in enumerate((2, 1, 1, 2)))
    index = torch.arange(3, device=gpu, dtype=torch.int32).expand(2, 1, 5, 3).contiguous()

    def f():
        return torch.autograd.grad(tokens.block_sparse_attention(q, k, v, index), (q, k, v), do)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = f()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in held]
        assert all(torch.equal(a, b) for a, b in zip(got, f()))


@gpu_only
def test_attention_of_a_cache_that_the_batch_shares(gpu):
    """Keys and values expanded over the batch (a stride of 0): the bits of their copies."""
    q = torch.randn(3, 70, 4, 64, device=gpu, requires_grad=True)
    cache = torch.randn(1, 200, 2, 64, device=gpu, requires_grad=True)
    index = torch.arange(4, device=gpu, dtype=torch.int32).expand(3, 2, 2, 4).contiguous()
    shared, copies = cache.expand(3, -1, -1, -1), cache.detach().repeat(3, 1, 1, 1).requires_grad_(True)
    outs = [tokens.block_sparse_attention(q, c, c, index) for c in (shared, copies)]
    assert torch.equal(*outs)
    do = torch.randn_like(outs[0])
    a = torch.autograd.grad(outs[0], (q, shared), do)
    b = torch.autograd.grad(outs[1], (q, copies), do)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


# ---- values and keys with a mean ------------------------------------------------------------


def query_gradient(q, k, v, do, scale):
    """(dq, how far off before it is rounded) in 64 bits, for any type. dp, delta and a score are sums of D 32-bit products, the score's
    exponent and logarithm off by 8 steps. p (for o, which delta is made of), o and ds are 32-bit numbers, or two pieces
    of 16 bits (bf16's keep 2^-16 of a value; n roundings of p, so six standard deviations of their sum); o and dq are sums over
    the n keys."""
    D, n, E, two = q.shape[1], k.shape[0], orc.E32, 2.0 ** -16
    x, dp = q @ k.T * scale, do @ v.T
    p = torch.softmax(x, -1)
    o = p @ v
    delta = (do * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    e_x = (D * (q.abs() @ k.abs().T) * abs(scale) + 8 * (1 + x.abs())) * E
    e_o = 6 * two * (p.square() @ v.square()).sqrt() + (p * 2 * e_x) @ v.abs() + n * E * (p @ v.abs()) + two * o.abs()
    e_delta = (do.abs() * e_o).sum(-1, keepdim=True) + D * E * (do.abs() * o.abs()).sum(-1, keepdim=True)
    e_ds = p * D * E * (do.abs() @ v.abs().T) + ds.abs() * (2 * e_x + two + (n + 4) * E)
    return ds @ k * scale, (e_ds @ k.abs() + e_delta * (p @ k).abs()) * abs(scale)


@gpu_only
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("key_mean,value_mean", [(0.0, 0.0), (3.0, 0.0), (0.0, 3.0), (1.0, 1.0), (3.0, 3.0)])
@pytest.mark.parametrize("L,Hq,block,n,D", [(256, 1, 64, 1024, 64), (40, 2, 32, 500, 32), (130, 1, 128, 900, 128), (16, 2, 64, 4000, 96)])
def test_query_gradients_of_keys_and_values_with_a_mean(gpu, t, key_mean, value_mean, L, Hq, block, n, D):
    """dq to its own rounding where every key and every value has a large part in common: none of it belongs in dq, and a rounding of
    o or of ds times that part would be larger than dq."""
    g = torch.Generator().manual_seed(n)
    km, vm = torch.randn(D, generator=g) * key_mean, torch.randn(D, generator=g) * value_mean
    q, k, v, do = ((torch.randn(1, m, h, D, generator=g) + a).to(t) for m, h, a in ((L, Hq, 0.0), (n, 1, km), (n, 1, vm), (L, Hq, 0.0)))
    blocks = -(-n // block)
    index = torch.arange(blocks, device=gpu, dtype=torch.int32).expand(1, 1, -(-L // block), blocks).contiguous()
    leaves = [x.to(gpu).requires_grad_(True) for x in (q, k, v)]
    (got,) = torch.autograd.grad(tokens.block_sparse_attention(*leaves, index, block=block), leaves[:1], do.to(gpu))
    for head in range(Hq):
        want, off = query_gradient(*(x[0, :, min(head, x.shape[2] - 1)].double() for x in (q, k, v, do)), D ** -0.5)
        h, dq = orc.half_step(t), got[0, :, head]
        orc.assert_within(dq, want, off + h * want.abs() + orc.tiny(t), "dq")
        # (roundings are spread evenly over a step: together at most 0.58 of the half step, that of a value just above a power of two)
        assert float((dq.double().cpu() - want).norm()) < 0.58 * h * float(want.norm()) + float(off.norm())
