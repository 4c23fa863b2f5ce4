"""The operators around attention together, as a layer uses them: normed and turned queries and keys
into windowed attention (training), the same layer decoding over a 4-bit cache, and both under CUDA
graphs and on other streams."""
import math

import pytest
import torch

import densecore_b200 as dc
from densecore_b200 import functional as F

pytestmark = pytest.mark.gpu


def layer(x, wqkv, wq, wk, pos, freq, h, kv, window, sinks):
    b, l, _ = x.shape
    d = wq.shape[0]
    y = x @ wqkv.T
    q = y[..., :h * d].view(b, l, h, d).transpose(1, 2)
    k = y[..., h * d:(h + kv) * d].view(b, l, kv, d).transpose(1, 2)
    v = y[..., (h + kv) * d:].view(b, l, kv, d).transpose(1, 2)
    q, k = F.qk_norm_rotary(q, k, wq, wk, pos, freq)
    return F.sliding_window_attention(q, k, v, window, sinks, enable_gqa=True).transpose(1, 2).reshape(b, l, h * d)


def plain(x, wqkv, wq, wk, pos, freq, h, kv, window, sinks):
    """The same layer in 64 bits."""
    x, wqkv, wq, wk = (t.double() for t in (x, wqkv, wq, wk))
    b, l, _ = x.shape
    d = wq.shape[0]
    y = x @ wqkv.T
    ang = pos[:, None].double() * freq
    rows = []
    for lo, n, w in ((0, h, wq), (h, kv, wk)):
        z = y[..., lo * d:(lo + n) * d].view(b, l, n, d).transpose(1, 2)
        z = z / (z.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
        a, c = z[..., :d // 2], z[..., d // 2:]
        rows.append(torch.cat((a * ang.cos() - c * ang.sin(), c * ang.cos() + a * ang.sin()), -1))
    v = y[..., (h + kv) * d:].view(b, l, kv, d).transpose(1, 2)
    q, k = rows
    k, v = (t.repeat_interleave(h // kv, 1) for t in (k, v))
    i, j = torch.arange(l, device="cuda")[:, None], torch.arange(l, device="cuda")
    vis = (j <= i) & ((i - j < window) | (j < sinks))
    p = torch.where(vis, q @ k.transpose(2, 3) / math.sqrt(d), -math.inf).softmax(-1)
    return (p @ v).transpose(1, 2).reshape(b, l, h * d)


def inputs(b=2, l=150, c=96, h=4, kv=2, d=64):
    g = torch.Generator(device="cuda").manual_seed(0)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")
    freq, _ = F.rotary_frequencies(d, device="cuda")
    return r(b, l, c), r((h + 2 * kv) * d, c) / math.sqrt(c), 1 + 0.2 * r(d), 1 + 0.2 * r(d), torch.arange(l, device="cuda"), freq


def test_layer_trains_as_the_formula():
    x, wqkv, wq, wk, pos, freq = inputs()
    args = (4, 2, 40, 4)
    ours = [t.clone().requires_grad_() for t in (x, wqkv, wq, wk)]
    refs = [t.double().requires_grad_() for t in (x, wqkv, wq, wk)]
    out, ref = layer(*ours, pos, freq, *args), plain(*refs, pos, freq, *args)
    go = torch.randn_like(out)
    got = torch.autograd.grad(out, ours, go)
    want = torch.autograd.grad(ref, refs, go.double())
    # The attention's 1e-5 bar, behind two fp32 products of 96 to 300 terms: 3e-5 of the largest value.
    for a, r in zip((out, *got), (ref, *want)):
        assert (a.double() - r).abs().max() <= 3e-5 * r.abs().max()


def test_decoding_over_the_cache_follows_the_full_sequence():
    # Token by token over the cache: the cache's own values, one layer, so the only difference to a
    # full pass over those values is the kernels' rounding.
    x, wqkv, wq, wk, pos, freq = inputs(b=3, l=70)
    h, kv, d, window, sinks = 4, 2, 64, 24, 2
    b, l, _ = x.shape
    y = x @ wqkv.T
    q = y[..., :h * d].view(b, l, h, d).transpose(1, 2)
    k = y[..., h * d:(h + kv) * d].view(b, l, kv, d).transpose(1, 2)
    v = y[..., (h + kv) * d:].view(b, l, kv, d).transpose(1, 2)
    cache = dc.KVCache4(3 * 5, kv, d, page_size=16)
    table = torch.randperm(15, device="cuda").to(torch.int32).view(3, 5)
    outs = []
    for t in range(l):
        at = torch.full((b,), t, dtype=torch.int32, device="cuda")
        qt, kt = F.qk_norm_rotary(q[:, :, t:t + 1], k[:, :, t:t + 1], wq, wk, at[:, None], freq)
        cache.append(kt, v[:, :, t:t + 1], table, at)
        outs.append(cache.attention(qt, table, at + 1, window=window, sinks=sinks))
    ck, cv = cache.read(table, torch.full((b,), l, dtype=torch.int32, device="cuda"), l)
    fq, fk = F.qk_norm_rotary(q, k, wq, wk, pos, freq)
    full = F.sliding_window_attention(fq, ck, cv, window, sinks, enable_gqa=True)
    got = torch.cat(outs, 2)
    assert (got - full).abs().max() <= 2e-5 * full.abs().max()
    # and the cache stands for the keys within half a scale (1/30 of a group's range, 2^-8 of its values)
    span = fk.unflatten(-1, (-1, 32)).amax(-1) - fk.unflatten(-1, (-1, 32)).amin(-1)
    bound = (span / 30 * 1.02 + 2.0 ** -7 * fk.abs().amax()).repeat_interleave(32, -1)
    assert ((ck - fk).abs() <= bound).all()


def test_training_step_replays_from_a_graph():
    x, wqkv, wq, wk, pos, freq = inputs(b=1, l=130)
    args = (4, 2, 33, 3)
    static = [t.clone().requires_grad_() for t in (x, wqkv, wq, wk)]
    go = torch.randn(1, 130, 256, device="cuda")

    def step():
        out = layer(*static, pos, freq, *args)
        return (out.detach(), *torch.autograd.grad(out, static, go))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for _ in range(3):
        with torch.no_grad():
            for t in static:
                t.copy_(torch.randn_like(t) * t.abs().mean())
            go.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step()))


def test_two_decode_graphs_and_eager_calls_between_them():
    cache = dc.KVCache4(64, 2, 128, page_size=16)
    table = torch.arange(64, device="cuda", dtype=torch.int32).view(2, 32)
    k = torch.randn(2, 2, 300, 128, device="cuda")
    cache.append(k, k, table, torch.zeros(2, dtype=torch.int32, device="cuda"))
    qs = [torch.randn(2, 8, 1, 128, device="cuda") for _ in range(2)]
    lens = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([300, 17], [250, 299])]

    def step(i):
        a = cache.attention(qs[i], table, lens[i])
        b = F.sliding_window_attention(qs[i], k, k, 100, 4, lengths=lens[i], enable_gqa=True)
        return a, b

    for i in range(2):
        step(i)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(step(i))
    for _ in range(3):
        for q in qs:
            q.normal_()
        graphs[0].replay()
        mid = step(1)
        graphs[1].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], step(i)))
        assert all(torch.equal(a, b) for a, b in zip(mid, outs[1]))
    # lengths are read at replay
    lens[0].copy_(torch.tensor([5, 6], dtype=torch.int32, device="cuda"))
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs[0], step(0)))


def test_two_streams_at_once():
    torch.manual_seed(0)
    sets = []
    for i in range(2):
        q = torch.randn(2, 4, 400, 64, device="cuda")
        sets.append((q, torch.randn(2, 4, 400, 64, device="cuda")))
    want = [F.sliding_window_attention(q, k, k, 50, 4) for q, k in sets]
    want1 = [F.sliding_window_attention(q[:, :, :1], k, k, 300, 4) for q, k in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                q, k = sets[i]
                got[i].append((F.sliding_window_attention(q, k, k, 50, 4), F.sliding_window_attention(q[:, :, :1], k, k, 300, 4)))
    torch.cuda.synchronize()
    for i in range(2):
        for a, b in got[i]:
            assert torch.equal(a, want[i]) and torch.equal(b, want1[i])
