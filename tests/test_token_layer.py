"""The view-token operators as they are used: a whole layer forward and backward against plain torch in 64 bits, in the
Gaussian head's training step, in captured graphs, on other streams, from two threads, and at sizes whose
offsets pass 32 bits."""
from __future__ import annotations

import math
import threading

import pytest
import torch

import token_oracle as orc

gpu_only = pytest.mark.gpu
BF16 = torch.bfloat16


def plain_layer(layer, x, positions, freqs, keep1, keep2, index, lengths=None):
    """ViewTokenLayer on host tensors in 64 bits, differentiable; the masks and the choice are given."""
    H, KV, D, block = layer.heads, layer.kv_heads, layer.dim, layer.block
    norm = lambda t, m: torch.nn.functional.layer_norm(t, t.shape[-1:], m.weight, m.bias, m.eps)  # noqa: E731
    B, L, _ = x.shape
    q, k, v = layer.qkv(norm(x, layer.norm1)).unflatten(-1, (-1, D)).split((H, KV, KV), 2)
    F, A = freqs.numel(), positions.shape[-1]
    angle = torch.stack([positions[:, i // (F // A)].double() * freqs[i] for i in range(F)], -1)[:, None]

    def turn(t):
        a, b = t[..., :F], t[..., F:2 * F]
        return torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), t[..., 2 * F:]], -1)

    q, k = turn(q), turn(k)
    see = torch.zeros(B, H, L, L, dtype=torch.bool)
    for b in range(B):
        n = L if lengths is None else int(lengths[b])
        for h in range(KV):
            for t in range(index.shape[2]):
                for j in index[b, h, t].tolist():
                    if j >= 0:
                        see[b, h * (H // KV):(h + 1) * (H // KV), t * block:min(n, (t + 1) * block), j * block:min(n, (j + 1) * block)] = True
    kh, vh = (t.repeat_interleave(H // KV, 2).permute(0, 2, 1, 3) for t in (k, v))
    s = (q.permute(0, 2, 1, 3) @ kh.transpose(-1, -2) / math.sqrt(D)).masked_fill(~see, -1e30)
    o = ((torch.softmax(s, -1) * see) @ vh).permute(0, 2, 1, 3).flatten(2)
    drop = lambda t, keep: torch.where(keep, t / (1 - layer.p), 0.0)  # noqa: E731
    s = x + drop(layer.out(o), keep1)
    return s + drop(layer.fc2(torch.nn.functional.gelu(layer.fc1(norm(s, layer.norm2)))), keep2), (q, k)


@gpu_only
@pytest.mark.parametrize("ragged", [False, True])
def test_layer_against_plain_torch(gpu, ragged):
    """f32 against 64 bits: some 12 operators, each within 64 * 2^-24 of its output's norm, and the norms' and the softmax's
    derivatives pass on at most about 4 times their input's error: 2e-4 of each result's norm."""
    import copy

    from my_depthsplat_amd import tokens as T
    from my_depthsplat_amd.token_layer import ViewTokenLayer
    torch.manual_seed(0)
    B, V, h, w, C = 2, 2, 9, 13, 48
    L = V * h * w
    layer = ViewTokenLayer(C, heads=3, top=3, p=0.2, block=32)
    ref = copy.deepcopy(layer).double()
    layer.to(gpu)
    pos, freqs = T.view_positions(V, h, w, gpu), T.rotary_frequencies(layer.part(2), 2, device=gpu)
    x64, dy64 = torch.randn(B, L, C, dtype=torch.float64).float().double(), torch.randn(B, L, C, dtype=torch.float64).float().double()
    lengths = torch.tensor([L, L - 50]) if ragged else None
    x = x64.float().to(gpu).requires_grad_(True)
    rng = T.dropout_rng(99, 4, gpu)
    y = layer(x, pos, freqs, rng, 6, None if lengths is None else lengths.to(gpu))
    grads = torch.autograd.grad(y, [x, *layer.parameters()], dy64.float().to(gpu))
    keep = [orc.keep_mask(B * L * C, 0.2, 99, 4, c).view(B, L, C) for c in (6, 7)]
    x64.requires_grad_(True)
    with torch.no_grad():  # the choice, from the same q and k in 64 bits
        q, k = plain_layer(ref, x64, pos.cpu(), freqs.cpu(), *keep, torch.full((B, 3, -(-L // 32), 1), -1), lengths)[1]
        index = orc.select_blocks(q, k, 3, 32, lengths, lengths)
    y64, _ = plain_layer(ref, x64, pos.cpu(), freqs.cpu(), *keep, index, lengths)
    grads64 = torch.autograd.grad(y64, [x64, *ref.parameters()], dy64)
    for name, a, b in zip(["y", "x", *(n for n, _ in ref.named_parameters())], (y, *grads), (y64, *grads64)):
        off = float((a.detach().double().cpu() - b.detach()).norm() / b.detach().norm())
        assert off < 2e-4, (name, off)


@gpu_only
def test_layer_in_bf16_and_refused_on_cpu(gpu):
    from my_depthsplat_amd import _lib
    from my_depthsplat_amd import tokens as T
    from my_depthsplat_amd.token_layer import ViewTokenLayer
    layer = ViewTokenLayer(64, heads=2, kv_heads=1).to(gpu, BF16).eval()
    pos, freqs = T.view_positions(1, 8, 9, gpu), T.rotary_frequencies(layer.part(2), 2, device=gpu)
    y = layer(torch.randn(2, 72, 64, device=gpu, dtype=BF16), pos, freqs)
    assert y.dtype == BF16 and bool(y.isfinite().all())
    with pytest.raises(_lib.DsplatError):
        layer.cpu()(torch.randn(2, 72, 64, dtype=BF16), pos.cpu(), freqs.cpu())


@pytest.mark.parametrize("kw", [dict(width=60, heads=2), dict(width=64, heads=0), dict(width=512, heads=2), dict(width=64, heads=4, kv_heads=3)])
def test_layer_refusals(kw):
    from my_depthsplat_amd.token_layer import ViewTokenLayer
    with pytest.raises(ValueError):
        ViewTokenLayer(**kw)


def test_head_without_token_layers_is_as_before():
    """No new parameters, buffers or random draws."""
    from my_depthsplat_amd.training import GaussianHead
    torch.manual_seed(0)
    a = GaussianHead(10, width=8, down=2)
    assert set(a.state_dict()) == {f"{m}.{p}" for m in ("stem", "body.1", "body.3", "out") for p in ("weight", "bias")}
    assert a(torch.rand(1, 2, 3, 8, 8), torch.rand(1, 2, 64, 1, 1)).shape == (1, 2, 64, 10)


@gpu_only
def test_head_with_token_layers_trains(gpu):
    """The training step runs through the layers: every parameter gets a finite gradient, the generator's step goes up, a
    second forward of the same step state gives the same result, and evaluation draws nothing."""
    from my_depthsplat_amd.training import GaussianHead
    torch.manual_seed(0)
    head = GaussianHead(10, width=24, down=2, token_layers=2, token_heads=2, token_top=2, token_dropout=0.1, seed=7).to(gpu)
    images, depths = torch.rand(2, 3, 3, 24, 16, device=gpu), torch.rand(2, 3, 24 * 16, 1, 1, device=gpu)
    state = head.rng.clone()
    y = head(images, depths)
    assert y.shape == (2, 3, 384, 10) and head.rng.tolist() == [7, 1]
    y.square().sum().backward()
    for n, p in head.named_parameters():
        assert p.grad is not None and bool(p.grad.isfinite().all()) and bool((p.grad != 0).any()), n
    z = head(images, depths)
    assert not torch.equal(y, z)
    head.rng.copy_(state)
    assert torch.equal(head(images, depths), y)
    head.eval()
    assert torch.equal(head(images, depths), head(images, depths)) and head.rng.tolist() == [7, 1]


def ops(gpu, seed):
    """name -> (static tensors, function of them): each operator forward and backward on tensors of its own."""
    from my_depthsplat_amd import tokens as T
    g = torch.Generator(device=gpu).manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device=gpu).to(BF16)  # noqa: E731
    leaf = lambda *s: r(*s).requires_grad_(True)  # noqa: E731
    rng = T.dropout_rng(seed, 1, gpu)
    freqs, pos = T.rotary_frequencies(64, device=gpu), torch.arange(200, device=gpu)
    out = {}
    x, res, w, b, dy, ds = leaf(300, 100), leaf(300, 100), leaf(100), leaf(100), r(300, 100), r(300, 100)
    out["norm"] = ((x, dy), lambda: (lambda y: (y, *torch.autograd.grad(y, (x, w, b), dy)))(T.layer_norm(x, w, b)))

    def fused():
        s, y = T.dropout_add_layer_norm(x, res, w, b, p=0.3, rng=rng, call=2)
        return (s, y, *torch.autograd.grad((s, y), (x, res, w, b), (ds, dy)))

    out["add_norm"] = ((x, res, dy, ds, rng), fused)
    out["dropout"] = ((x, dy, rng), lambda: (lambda y: (y, *torch.autograd.grad(y, x, dy)))(T.dropout(x, 0.4, rng)))
    q, k, v, do = leaf(2, 200, 4, 64), leaf(2, 200, 2, 64), leaf(2, 200, 2, 64), r(2, 200, 4, 64)
    out["rotary"] = ((q, k, do), lambda: (lambda t: (*t, *torch.autograd.grad(t[0], q, do)))(T.rotary(q, k, pos, freqs)))
    lens = torch.tensor([200, 150], device=gpu, dtype=torch.int32)

    def attend():
        index = T.select_blocks(q, k, 2, block=32, kv_lengths=lens)
        o = T.block_sparse_attention(q, k, v, index, block=32, kv_lengths=lens)
        return (index, o, *torch.autograd.grad(o, (q, k, v), do))

    out["attend"] = ((q, k, v, do, lens), attend)
    one = r(2, 1, 4, 64)

    def few():
        with torch.no_grad():
            return (T.block_sparse_attention(one, k, v, index1),)

    index1 = torch.tensor([[[[0, 1, 2, 3] * 5]] * 2] * 2, dtype=torch.int32, device=gpu)
    out["few"] = ((one, k, v), few)
    return out


@gpu_only
@pytest.mark.parametrize("name", ["norm", "add_norm", "dropout", "rotary", "attend", "few"])
def test_captured_and_replayed(gpu, name):
    """Two graphs of the operator, replayed in turn on inputs that change, with eager work between: each replay is the eager
    result, bit for bit."""
    calls = [ops(gpu, s)[name] for s in (1, 2)]
    graphs = []
    for _, f in calls:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = f()
        graphs.append((graph, held))
    for turn in range(3):
        for (tensors, f), (graph, held) in zip(calls, graphs):
            with torch.no_grad():
                for t in tensors:
                    if t.is_floating_point():
                        t.copy_(torch.randn(t.shape, device=gpu))
                    elif t.dtype == torch.int64:
                        t[1] += 1
                    else:
                        t.sub_(7)
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in held]
            for a, e in zip(got, f()):
                assert torch.equal(a, e), (name, turn)


@gpu_only
def test_captured_backward_of_lists_that_change(gpu):
    """Two graphs whose key blocks' lists, and so the parts of dk and dv that are worked off by themselves, differ at every replay."""
    from my_depthsplat_amd import tokens as T
    r = lambda *s: torch.randn(*s, device=gpu).to(BF16)  # noqa: E731
    calls, graphs = [], []
    for _ in range(2):
        q, k, v, do = r(2, 1900, 2, 32).requires_grad_(True), r(2, 700, 1, 32).requires_grad_(True), r(2, 700, 1, 32).requires_grad_(True), r(2, 1900, 2, 32)
        index = torch.zeros(2, 1, 60, 5, dtype=torch.int32, device=gpu)

        def f(q=q, k=k, v=v, do=do, index=index):
            return torch.autograd.grad(T.block_sparse_attention(q, k, v, index, block=32), (q, k, v), do)

        calls.append((index, f))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            f()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = f()
        graphs.append((graph, held))
    for turn in range(4):
        for (index, f), (graph, held) in zip(calls, graphs):
            index.copy_(torch.randint(-3, 22, index.shape, device=gpu))
            index[:, :, :, 0] = 5 * turn  # a popular block, another one each time
            graph.replay()
            torch.cuda.synchronize()
            got = [t.clone() for t in held]
            assert all(torch.equal(a, e) for a, e in zip(got, f())), turn


@gpu_only
@pytest.mark.parametrize("name", ["norm", "add_norm", "dropout", "rotary", "attend", "few"])
def test_on_another_stream_and_from_two_threads(gpu, name):
    calls = [ops(gpu, s)[name] for s in (3, 4)]
    want = [[t.clone() for t in f()] for _, f in calls]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for (_, f), w in zip(calls, want):
            assert all(torch.equal(a, b) for a, b in zip(f(), w))
    torch.cuda.current_stream().wait_stream(side)
    failed = []

    def work(f, w, stream):
        try:
            with torch.cuda.stream(stream):
                for _ in range(20):
                    if not all(torch.equal(a, b) for a, b in zip(f(), w)):
                        failed.append(name)
        except Exception as e:  # noqa: BLE001
            failed.append(repr(e))

    threads = [threading.Thread(target=work, args=(f, w, torch.cuda.Stream())) for (_, f), w in zip(calls, want)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed


@gpu_only
def test_offsets_past_32_bits(gpu):
    """Caches, rows and elements whose offsets pass 2^31 and 2^32 give what their last part alone gives."""
    from my_depthsplat_amd import tokens as T
    if torch.cuda.get_device_properties(gpu).total_memory < 64 << 30:
        pytest.skip("needs 64 GB")
    L = 17_500_000  # x 128 channels: 2.24e9 elements
    k = torch.zeros(1, L, 1, 128, device=gpu, dtype=BF16)
    k[:, -200:] = torch.randn(1, 200, 1, 128, device=gpu)
    q = torch.randn(1, 64, 1, 128, device=gpu).to(BF16)
    blocks = -(-L // 64)
    index = torch.tensor([[[[0, blocks - 3, blocks - 2, blocks - 1]]]], dtype=torch.int32, device=gpu)
    lo = (blocks - 3) * 64
    short = torch.cat([k[:, :64], k[:, lo:]], 1)
    leaves = [q.requires_grad_(True), short.requires_grad_(True)]
    o = T.block_sparse_attention(q, short, short, torch.arange(4, device=gpu, dtype=torch.int32).view(1, 1, 1, 4))
    want = torch.autograd.grad(o, leaves, torch.ones_like(o))
    k.requires_grad_(True)
    long = T.block_sparse_attention(q, k, k, index)
    assert torch.equal(long, o)
    dq, dk = torch.autograd.grad(long, (q, k), torch.ones_like(long))
    assert torch.equal(dq, want[0]) and torch.equal(dk[:, lo:], want[1][:, 64:]) and torch.equal(dk[:, :64], want[1][:, :64])
    assert not bool(dk[:, 64:lo].any())
    del dk, long
    with torch.no_grad():
        qm = k[:, lo + 64:lo + 128].float().mean(1, keepdim=True).expand(1, 64, 1, 128).to(BF16)
        assert blocks - 2 in T.select_blocks(qm, k, 2).flatten().tolist()
        x = k.view(-1, 128)
        assert torch.equal(T.layer_norm(x)[-200:], T.layer_norm(x[-200:].contiguous()))
        freqs, pos = T.rotary_frequencies(128, device=gpu), torch.arange(L, device=gpu)
        assert torch.equal(T.rotary(k, None, pos, freqs)[0][:, -200:], T.rotary(k[:, -200:], None, pos[-200:], freqs)[0])
    del k, x, short, leaves, want
    n = 2 ** 32 + 2 ** 20 + 6
    y = T.dropout(torch.ones(n, device=gpu, dtype=BF16), 0.5, T.dropout_rng(11, 3, gpu), 9)
    for at in (0, 2 ** 31, 2 ** 32, n - 6):
        group = at // 4
        words = orc.philox4x32((group & 0xFFFFFFFF, group >> 32, 9, 3), (11, 0))[at % 4:]
        assert (y[at:at + len(words)] != 0).tolist() == [w >= 2 ** 31 for w in words]
