"""Sliding-window attention against the formula in 64 bits.

Tolerance: the bar of the other attention kernels, max|delta| <= 1e-5 max|ref| (3xTF32 products are off
by about 2^-21 of their absolute terms, the fp32 kernels by less; scores here stay below 10, so weights
are off by a few 1e-6). Single-pass TF32 rounds operands to 11 bits: 2^-11 of the absolute terms of a
score, sums of D products of random sign; 1e-2."""
import math

import pytest
import torch

import densecore_b200 as dc
from densecore_b200 import functional as F

pytestmark = pytest.mark.gpu


def reference(q, k, v, window, sinks, offset, mask=None, lens=None, scale=None):
    q, k, v = q.double(), k.double(), v.double()
    h, kv = q.shape[1], k.shape[1]
    k, v = (t.repeat_interleave(h // kv, 1) for t in (k, v))
    s = q @ k.transpose(2, 3) * (1 / math.sqrt(q.shape[3]) if scale is None else scale)
    i, j = torch.arange(q.shape[2], device="cuda")[:, None], torch.arange(k.shape[2], device="cuda")
    t = (i + offset)[None] if lens is None else (lens.clamp(0, k.shape[2]).long() - 1)[:, None, None]
    vis = (j <= t) & ((t - j < window) | (j < sinks))
    vis = vis[:, None]
    if mask is not None:
        if mask.dtype == torch.bool:
            vis = vis & mask
        else:
            vis = vis & (mask > -1e30)
            s = s + mask.clamp_min(-1e30).double()
    s = torch.where(vis, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    return (p / torch.where(total == 0, 1.0, total)) @ v


def rel(got, ref):
    assert torch.isfinite(got).all()
    scale = ref.abs().max().item() if ref.numel() else 0.0
    return (got.double() - ref).abs().max().item() / (scale or 1.0) if ref.numel() else 0.0


def make(b, h, kv, l, s, d, layout, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *x: torch.randn(x, generator=g, device="cuda")
    if layout == "bshd":
        return r(b, l, h, d).transpose(1, 2), r(b, s, kv, d).transpose(1, 2), r(b, s, kv, d).transpose(1, 2)
    if layout == "odd":  # no TMA: rows at odd strides
        return r(b, h, l, d + 1)[..., 1:], r(b, kv, s, d + 1)[..., 1:], r(b, kv, s, d + 3)[..., :d]
    return r(b, h, l, d), r(b, kv, s, d), r(b, kv, s, d)


def check(q, k, v, window, sinks, offset=None, mask=None, tol=1e-5, scale=None):
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = F.sliding_window_attention(*leaves, window, sinks, attn_mask=mask, offset=offset, scale=scale, enable_gqa=True)
    go = torch.randn(out.shape, device="cuda")
    grads = torch.autograd.grad(out, leaves, go)
    refs = [t.detach().double().requires_grad_() for t in (q, k, v)]
    ro = reference(*refs, window, sinks, k.shape[2] - q.shape[2] if offset is None else offset, mask, scale=scale)
    rg = torch.autograd.grad(ro, refs, go.double())
    for name, a, r in zip(("out", "dq", "dk", "dv"), (out, *grads), (ro, *rg)):
        assert rel(a.detach(), r.detach()) <= tol, (name, rel(a.detach(), r.detach()))
    assert dc._lib.load().dc_device_status(1) == 0
    return out.detach(), grads


CASES = [  # b, h, kv, l, s, d, window, sinks, offset
    (1, 1, 1, 1, 1, 64, 1, 0, None), (2, 3, 3, 17, 17, 64, 5, 2, None), (1, 2, 2, 129, 129, 64, 64, 0, None),
    (2, 4, 2, 300, 300, 64, 33, 4, None), (1, 2, 1, 257, 257, 128, 100, 1, None), (1, 2, 2, 640, 640, 64, 128, 130, None),
    (1, 2, 2, 100, 700, 64, 200, 3, None), (1, 1, 1, 64, 1000, 128, 1, 1, None), (2, 2, 2, 200, 90, 64, 20, 2, None),
    (1, 2, 2, 200, 200, 64, 20, 2, 0), (1, 2, 2, 150, 150, 128, 40, 0, 70), (1, 2, 2, 150, 150, 64, 40, 5, -60),
    (1, 1, 1, 50, 50, 64, 10, 2, -200), (1, 1, 1, 50, 50, 64, 10, 2, 400), (1, 1, 1, 50, 50, 64, 10, 0, 400),
    (1, 2, 2, 130, 130, 64, 10 ** 12, 0, None), (1, 1, 1, 130, 130, 64, 7, 10 ** 12, None), (1, 8, 1, 70, 333, 64, 90, 64, None),
    (1, 2, 2, 40, 40, 32, 9, 3, None), (1, 2, 1, 75, 130, 20, 17, 40, None), (1, 1, 1, 33, 70, 256, 12, 3, None),
    (1, 2, 2, 1, 500, 64, 100, 4, None), (2, 4, 2, 1, 500, 128, 100, 4, None), (1, 2, 2, 1, 500, 64, 100, 4, 700),
    (1, 2, 2, 1, 500, 64, 100, 4, 520), (1, 2, 1, 1, 500, 64, 100, 4, -3), (1, 2, 1, 1, 500, 64, 100, 0, 499)]


@pytest.mark.parametrize("layout", ["plain", "bshd", "odd"])
@pytest.mark.parametrize("case", CASES)
def test_forward_and_backward(case, layout):
    b, h, kv, l, s, d, window, sinks, offset = case
    check(*make(b, h, kv, l, s, d, layout), window, sinks, offset)


@pytest.mark.parametrize("d", [64, 128, 48])
@pytest.mark.parametrize("kind", ["padding", "left", "rows", "bias", "lowest", "inf", "full"])
def test_masks(kind, d):
    b, h, s = 2, 4, 200
    q, k, v = make(b, h, 2, s, s, d, "bshd", 3)
    j = torch.arange(s, device="cuda")
    mask = {
        "padding": lambda: (j < torch.tensor([150, 60], device="cuda")[:, None])[:, None, None],
        "left": lambda: (j >= torch.tensor([150, 0], device="cuda")[:, None])[:, None, None],  # empty first rows
        "rows": lambda: (torch.arange(s, device="cuda") % 3 != 0)[:, None].expand(s, s),  # every third row empty
        "bias": lambda: torch.randn(1, h, s, s, device="cuda"),
        "lowest": lambda: torch.where(j % 2 == 0, torch.finfo(torch.float32).min, 0.5).expand(1, 1, s, s).clone(),
        "inf": lambda: torch.where(j < 120, -math.inf, 0.0).expand(s, s).clone(),
        "full": lambda: torch.rand(b, h, s, s, device="cuda") < 0.5,
    }[kind]()
    out, grads = check(q, k, v, 40, 0 if kind in ("inf", "left") else 4, mask=mask)
    if kind == "rows":
        assert (out[:, :, ::3] == 0).all() and (grads[0][:, :, ::3] == 0).all()
    if kind == "lowest":  # a row of lowest values only sees nothing: row 0 of a window of one
        low = torch.full((s, s), torch.finfo(torch.float32).min, device="cuda")
        assert (F.sliding_window_attention(q, k, v, 40, 4, attn_mask=low, enable_gqa=True) == 0).all()


@pytest.mark.parametrize("d", [64, 128, 32])
def test_hidden_keys_may_hold_anything(d):
    # Infinities and NaN in keys that a bool or -inf mask hides do not reach the scores; masked values
    # must be finite.
    s = 150
    q, k, v = make(1, 2, 2, s, s, d, "plain", 4)
    hide = torch.zeros(s, dtype=torch.bool, device="cuda")
    hide[10:30] = True
    bad = k.clone()
    bad[:, :, 10:20], bad[:, :, 20:30] = math.nan, math.inf
    clean = F.sliding_window_attention(q, k, v, 50, 4, attn_mask=~hide.expand(s, s))
    assert torch.equal(F.sliding_window_attention(q, bad, v, 50, 4, attn_mask=~hide.expand(s, s)), clean)
    minus = torch.where(hide, -math.inf, 0.0).expand(s, s).clone()
    assert rel(F.sliding_window_attention(q, bad, v, 50, 4, attn_mask=minus), clean.double()) <= 1e-6


def test_long_windows_take_the_one_tile_kernel():
    # window + tile + sinks over 64 key blocks at head dim 128
    q, k, v = make(1, 1, 1, 4000, 4000, 128, "bshd", 5)
    check(q, k, v, 2500, 4)
    q, k, v = make(1, 2, 2, 6000, 6000, 64, "bshd", 6)
    check(q, k, v, 5000, 70)


def test_whole_window_is_causal_attention():
    q, k, v = make(2, 3, 3, 333, 333, 64, "bshd", 7)
    causal = dc.scaled_dot_product_attention(q, k, v, is_causal=True)
    assert torch.equal(F.sliding_window_attention(q, k, v, 333), causal)


@pytest.mark.parametrize("mode,tol", [("fp32", 1e-5), ("tf32", 1e-2)])
def test_precisions(mode, tol):
    dc.set_sdpa_precision(mode)
    try:
        for d in (64, 128):
            check(*make(1, 2, 1, 200, 260, d, "bshd", 8), 64, 3, tol=tol)
    finally:
        dc.set_sdpa_precision(None)


def test_negative_and_zero_scale():
    q, k, v = make(1, 2, 2, 140, 140, 64, "bshd", 9)
    for scale in (-0.2, 0.0, 1.0):
        check(q, k, v, 30, 2, scale=scale)


@pytest.mark.parametrize("d", [64, 128, 40])
@pytest.mark.parametrize("heads", [(4, 4), (4, 2), (8, 2), (12, 4), (8, 1), (5, 1)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (64, 4), (700, 100), (10 ** 6, 0)])
def test_single_token_with_lengths(d, heads, window, sinks):
    h, kv = heads
    s = 777
    lens = torch.tensor([0, 1, 5, 64, 300, 776, 777, 12], dtype=torch.int32, device="cuda")
    b = len(lens)
    q, k, v = make(b, h, kv, 1, s, d, "plain", 11)
    for i, n in enumerate(lens.tolist()):  # what lies behind a sequence's end is never used
        k[i, :, n:], v[i, :, n:] = math.nan, math.nan
    got = F.sliding_window_attention(q, k, v, window, sinks, lengths=lens, enable_gqa=True)
    ref = reference(q, torch.nan_to_num(k), torch.nan_to_num(v), window, sinks, 0, lens=lens)
    assert rel(got, ref) <= 1e-5
    assert (got[0] == 0).all()
    strided = F.sliding_window_attention(q, k, v, window, sinks, lengths=lens.repeat_interleave(3)[::3], enable_gqa=True)
    assert torch.equal(strided, got)


@pytest.mark.parametrize("d", [64, 128])
def test_single_token_masks_and_batch_of_one(d):
    q, k, v = make(1, 8, 2, 1, 5000, d, "bshd", 12)
    ref = reference(q, k, v, 3000, 8, 4999)
    got = F.sliding_window_attention(q, k, v, 3000, 8, enable_gqa=True)
    assert rel(got, ref) <= 1e-5
    bias = torch.randn(1, 8, 1, 5000, device="cuda")
    assert rel(F.sliding_window_attention(q, k, v, 3000, 8, attn_mask=bias, enable_gqa=True),
               reference(q, k, v, 3000, 8, 4999, bias)) <= 1e-5
    hide = (torch.arange(5000, device="cuda") < 4990)
    assert rel(F.sliding_window_attention(q, k, v, 5, 0, attn_mask=hide.view(1, 1, 1, -1), enable_gqa=True),
               reference(q, k, v, 5, 0, 4999, hide.view(1, 1, 1, -1))) == 0.0  # a row that sees nothing
    low = torch.full((1, 1, 1, 5000), torch.finfo(torch.float32).min, device="cuda")
    low[..., 4999] = 0
    assert rel(F.sliding_window_attention(q, k, v, 100, 4, attn_mask=low, enable_gqa=True),
               reference(q, k, v, 100, 4, 4999, low)) <= 1e-5
    lse = dc._native._sliding_window(q, k, v, 3000, 8, 4999)[1]
    x = (q.double().view(2, 4, d) @ k[0].double().transpose(1, 2)) / math.sqrt(d)
    x = torch.cat((x[..., :8], x[..., 2000:]), -1)
    assert (lse.view(2, 4).double() - x.logsumexp(-1)).abs().max() <= 1e-5


def test_rank_three_and_empty():
    q = torch.randn(2, 9, 64, device="cuda")
    got = F.sliding_window_attention(q, q, q, 4, 1)
    assert rel(got[:, None], reference(q[:, None], q[:, None], q[:, None], 4, 1, 0)) <= 1e-5
    for shape_q, shape_k in (((0, 2, 3, 64), (0, 2, 3, 64)), ((1, 2, 0, 64), (1, 2, 5, 64)), ((1, 2, 4, 64), (1, 2, 0, 64)),
                             ((1, 2, 1, 64), (1, 2, 0, 64))):
        a, c = torch.randn(shape_q, device="cuda", requires_grad=True), torch.randn(shape_k, device="cuda", requires_grad=True)
        y = F.sliding_window_attention(a, c, c, 3, 1)
        y.sum().backward()
        assert y.shape == a.shape and (y == 0).all() and (c.grad == 0).all()


def test_repeats_bit_for_bit():
    q, k, v = make(2, 4, 2, 500, 500, 64, "bshd", 13)
    first = check(q, k, v, 60, 4)[0]
    for _ in range(3):
        assert torch.equal(F.sliding_window_attention(q, k, v, 60, 4, enable_gqa=True), first)


@pytest.mark.parametrize("layout", ["bshd", "odd"])
@pytest.mark.parametrize("case", [  # b, h, kv, l, s, d, window, sinks, offset
    (1, 1, 1, 1500, 1500, 64, 30, 4, None), (1, 4, 2, 1100, 1300, 64, 17, 200, None), (1, 2, 1, 1000, 1000, 128, 40, 130, None),
    (2, 2, 2, 2000, 2000, 64, 1, 1, None), (1, 1, 1, 1500, 700, 64, 30, 4, -300), (1, 1, 1, 1300, 1300, 64, 30, 5000, None)])
def test_first_tokens_seen_by_many_rows(case, layout):
    # The first tokens' gradients are summed over runs of far rows by CTAs of their own.
    b, h, kv, l, s, d, window, sinks, offset = case
    q, k, v = make(b, h, kv, l, s, d, layout, 14)
    check(q, k, v, window, sinks, offset)
    mask = torch.arange(s, device="cuda") % 5 != 0
    check(q, k, v, window, sinks, offset, mask=mask.view(1, 1, 1, s))
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    go = torch.ones(b, h, l, d, device="cuda")
    runs = [torch.autograd.grad(F.sliding_window_attention(*leaves, window, sinks, offset=offset, enable_gqa=True), leaves, go)
            for _ in range(2)]
    assert all(torch.equal(x, y) for x, y in zip(*runs))


@pytest.mark.parametrize("layout", ["plain", "bshd"])
@pytest.mark.parametrize("dims", [(4, 4), (20, 20), (32, 32), (48, 80), (80, 48), (96, 96), (128, 32), (30, 30), (33, 64), (124, 128), (160, 64), (200, 256)])
def test_head_dims(dims, layout):
    e, ev = dims
    g = torch.Generator(device="cuda").manual_seed(15)
    r = lambda *x: torch.randn(x, generator=g, device="cuda")
    if layout == "bshd":
        q, k, v = r(2, 170, 4, e).transpose(1, 2), r(2, 200, 2, e).transpose(1, 2), r(2, 200, 2, ev).transpose(1, 2)
    else:
        q, k, v = r(2, 4, 170, e), r(2, 2, 200, e), r(2, 2, 200, ev)
    check(q, k, v, 50, 3)
    check(q, k, v, 50, 3, mask=torch.rand(2, 1, 170, 200, device="cuda") < 0.7)
    # many rows behind the first tokens
    q, k, v = r(1, 2, 1200, e), r(1, 1, 1200, e), r(1, 1, 1200, ev)
    check(q, k, v, 20, 3)


@pytest.mark.parametrize("d", [4, 32, 36, 80, 96, 160, 256, 33])
def test_single_token_head_dims(d):
    lens = torch.tensor([300, 1, 0, 299], dtype=torch.int32, device="cuda")
    q, k, v = make(4, 6, 2, 1, 300, d, "plain", 16)
    for i, n in enumerate(lens.tolist()):
        k[i, :, n:], v[i, :, n:] = math.nan, math.nan
    got = F.sliding_window_attention(q, k, v, 100, 5, lengths=lens, enable_gqa=True)
    assert rel(got, reference(q, torch.nan_to_num(k), torch.nan_to_num(v), 100, 5, 0, lens=lens)) <= 1e-5


def test_ragged_single_tokens_with_masks():
    lens = torch.tensor([300, 1, 0, 150], dtype=torch.int32, device="cuda")
    q, k, v = make(4, 4, 2, 1, 300, 64, "plain", 17)
    bias = torch.randn(4, 1, 1, 300, device="cuda")
    hide = torch.rand(4, 4, 1, 300, device="cuda") < 0.5
    for mask in (bias, hide):
        got = F.sliding_window_attention(q, k, v, 100, 5, attn_mask=mask, lengths=lens, enable_gqa=True)
        assert rel(got, reference(q, k, v, 100, 5, 0, mask, lens=lens)) <= 1e-5


def test_broadcast_keys_get_summed_gradients():
    # Keys and values shared by every sequence of the batch: views without a batch stride.
    q = torch.randn(3, 2, 90, 64, device="cuda", requires_grad=True)
    k = torch.randn(1, 2, 90, 64, device="cuda", requires_grad=True)
    v = torch.randn(1, 2, 90, 64, device="cuda", requires_grad=True)
    out = F.sliding_window_attention(q, k.expand(3, -1, -1, -1), v.expand(3, -1, -1, -1), 20, 2)
    go = torch.randn_like(out)
    got = torch.autograd.grad(out, (q, k, v), go)
    refs = [t.detach().double().requires_grad_() for t in (q, k, v)]
    ro = reference(refs[0], refs[1].expand(3, -1, -1, -1), refs[2].expand(3, -1, -1, -1), 20, 2, 0)
    for a, r in zip((out, *got), (ro, *torch.autograd.grad(ro, refs, go.double()))):
        assert rel(a.detach(), r.detach()) <= 1e-5


def test_long_cache_past_two_to_the_32_bytes():
    if torch.cuda.get_device_properties(0).total_memory < 60 << 30:
        pytest.skip("needs memory")
    s = 9_000_000  # 4.6 GB each
    k = torch.zeros(1, 1, s, 128, device="cuda")
    v = torch.zeros(1, 1, s, 128, device="cuda")
    k[:, :, -200:].normal_(), v[:, :, -200:].normal_(), k[:, :, :4].normal_(), v[:, :, :4].normal_()
    q = torch.randn(1, 2, 1, 128, device="cuda")
    got = F.sliding_window_attention(q, k, v, 150, 4, enable_gqa=True)
    kk, vv = (torch.cat((t[:, :, :4], t[:, :, -150:]), 2) for t in (k, v))
    assert rel(got, reference(q, kk, vv, 1000, 0, 153)) <= 1e-5
    two = F.sliding_window_attention(torch.cat((q, q), 2), k, v, 150, 4, enable_gqa=True)[:, :, 1:]
    assert rel(two, reference(q, kk, vv, 1000, 0, 153)) <= 1e-5


# ---- long windows at head dims above 64: pairs of fp16 (22 bits, rounded to nearest, at most 2^-22 of an
# operand, so a few 2^-22 of a score's absolute terms), tighter than the TF32 pairs of the bar above.
def ran(f):
    """The kernels that f() launched."""
    dc._lib.kernel_timing(True)
    dc._lib.kernel_timing_report(True)
    f()
    torch.cuda.synchronize()
    names = set(dc._lib.kernel_timing_report(True))
    dc._lib.kernel_timing(False)
    return names


LONG = [  # b, h, kv, l, s, e, ev, window, sinks, offset
    (1, 2, 2, 1400, 1400, 128, 128, 10 ** 12, 0, None), (2, 2, 2, 2000, 2000, 128, 128, 700, 4, None),
    (1, 4, 1, 700, 700, 128, 128, 333, 0, None), (1, 4, 2, 900, 900, 96, 128, 800, 70, None),
    (1, 2, 2, 1283, 1283, 68, 100, 1283, 3, None), (1, 2, 2, 1301, 1301, 128, 4, 1200, 0, None),
    (1, 8, 1, 129, 1999, 128, 128, 1500, 5, None), (1, 8, 1, 37, 640, 80, 80, 600, 0, None),
    (1, 4, 1, 128, 704, 128, 128, 700, 1, 500), (1, 2, 2, 1500, 1500, 128, 128, 1400, 0, 300),
    (1, 8, 1, 2, 65, 128, 128, 10 ** 12, 0, 4000), (1, 3, 1, 1100, 1100, 72, 124, 1000, 900, None),
    (1, 4, 1, 900, 900, 128, 128, 633, 1, None), (1, 32, 1, 37, 640, 80, 80, 600, 0, None),
    (1, 8, 1, 128, 704, 128, 128, 700, 1, 500), (1, 64, 1, 70, 300, 128, 128, 280, 2, None)]


def pays(l, s, h, kv, window, offset):
    """Whether a mean row sees 192 keys and 384 more per key row that is packed for it."""
    first = (s - l if offset is None else offset) + 1
    mean = sum(min(first + i, window, s) for i in range(l)) / l
    return mean * l * h >= 192 * l * h + 384 * s * kv


@pytest.mark.parametrize("layout", ["plain", "bshd"])
@pytest.mark.parametrize("case", LONG)
def test_long_windows_above_64_columns(case, layout):
    b, h, kv, l, s, e, ev, window, sinks, offset = case
    q, k, v = make(b, h, kv, l, s, 128, layout, 20)
    q, k, v = q[..., :e], k[..., :e], v[..., :ev]
    names = ran(lambda: F.sliding_window_attention(q, k, v, window, sinks, offset=offset, enable_gqa=True))
    assert ("window_attend" in names) == pays(l, s, h, kv, window, offset)
    check(q, k, v, window, sinks, offset)


@pytest.mark.parametrize("kind", ["padding", "left", "rows", "bias", "lowest", "full", "strided"])
def test_long_windows_masks(kind):
    b, h, s = 2, 2, 1400
    q, k, v = make(b, h, h, s, s, 128, "bshd", 21)
    j = torch.arange(s, device="cuda")
    mask = {
        "padding": lambda: (j < torch.tensor([1300, 60], device="cuda")[:, None])[:, None, None],
        "left": lambda: (j >= torch.tensor([700, 0], device="cuda")[:, None])[:, None, None],  # empty first rows
        "rows": lambda: (j % 3 != 0)[:, None].expand(s, s),  # every third row empty
        "bias": lambda: torch.randn(1, h, s, s, device="cuda"),
        "lowest": lambda: torch.where(j % 2 == 0, torch.finfo(torch.float32).min, 0.5).expand(1, 1, s, s).clone(),
        "full": lambda: torch.rand(b, h, s, s, device="cuda") < 0.5,
        "strided": lambda: torch.randn(s, 2 * s + 1, device="cuda")[:, 1::2],
    }[kind]()
    call = lambda: F.sliding_window_attention(q, k, v, 1300, 2, attn_mask=mask)
    assert "window_attend" in ran(call)
    out, grads = check(q, k, v, 1300, 0 if kind == "left" else 2, mask=mask)
    if kind == "rows":
        assert (out[:, :, ::3] == 0).all() and (grads[0][:, :, ::3] == 0).all()
    if kind == "lowest":
        low = torch.full((s, s), torch.finfo(torch.float32).min, device="cuda")
        assert (F.sliding_window_attention(q, k, v, 1300, attn_mask=low) == 0).all()


def test_long_windows_hidden_keys_may_hold_anything():
    s = 1400
    q, k, v = make(1, 2, 2, s, s, 128, "plain", 22)
    hide = torch.zeros(s, dtype=torch.bool, device="cuda")
    hide[10:30] = True
    hide[640:704] = True  # a whole tile of keys
    bad = k.clone()
    bad[:, :, 10:20], bad[:, :, 20:30], bad[:, :, 640:704] = math.nan, math.inf, math.nan
    clean = F.sliding_window_attention(q, k, v, 1300, 4, attn_mask=~hide.expand(s, s))
    assert rel(F.sliding_window_attention(q, bad, v, 1300, 4, attn_mask=~hide.expand(s, s)), clean.double()) <= 1e-6
    minus = torch.where(hide, -math.inf, 0.0).expand(s, s).clone()
    assert rel(F.sliding_window_attention(q, bad, v, 1300, 4, attn_mask=minus), clean.double()) <= 1e-6


@pytest.mark.parametrize("big", [1e3, 1e6, 1e10, 1e30])
@pytest.mark.parametrize("what", ["key", "value", "key column", "value column", "value tile", "small values"])
def test_long_windows_outliers_leave_other_rows_exact(what, big):
    # One key, value, column or tile far larger than the rest: rows that do not see it, or columns beside
    # it, keep the tolerance relative to their own size. (The oracle's rows that see a huge key have one
    # weight of 1; their scores' errors are relative to the huge one and are not compared.)
    s, w = 2100, 800
    q, k, v = make(1, 2, 2, s, s, 128, "plain", 23)
    if what == "key":
        k[:, :, 100] *= big
    elif what == "value":
        v[:, :, 100] *= big
    elif what == "key column":  # seen by queries that have nothing in that column
        k[..., 5] *= big
        q[..., 5] = 0
    elif what == "value column":
        v[..., 5] *= big
    elif what == "value tile":
        v[:, :, 64:128] *= big
    else:
        v[:, :, 101:] /= big
    out = F.sliding_window_attention(q, k, v, w)
    ref = reference(q, k, v, w, 0, 0)
    rows, cols = slice(100 + w, s), [c for c in range(128) if c != 5]
    if what in ("key column", "value column"):
        rows = slice(0, s)
    assert rel(out[:, :, rows][..., cols], ref[:, :, rows][..., cols]) <= 1e-5
    assert dc._lib.load().dc_device_status(1) == 0


@pytest.mark.parametrize("scale", [1e-30, 1e-18, 1e18, 1e30])
def test_long_windows_of_any_magnitude(scale):
    # Powers of ten that leave the scores where they were, and values of any size.
    s = 1300
    q, k, v = make(1, 2, 2, s, s, 128, "plain", 24)
    assert rel(F.sliding_window_attention(q * scale, k / scale, v * scale, s), reference(q * scale, k / scale, v * scale, s, 0, 0)) <= 1e-5


def test_long_windows_of_zeros():
    s = 1300
    q, k, v = make(1, 2, 2, s, s, 128, "plain", 25)
    q[:, :, 5] = 0
    k[:, :, 64:192] = 0
    v[:, :, 128:300] = 0
    v[..., 7] = 0
    check(q, k, v, s, 0)
    assert (F.sliding_window_attention(q, k, torch.zeros_like(v), s) == 0).all()


def test_long_windows_captured_and_on_two_streams():
    s = 1400
    q, k, v = make(1, 2, 2, s, s, 128, "plain", 26)
    f = lambda: F.sliding_window_attention(q, k, v, 1300, 2)
    first = f()
    f()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = f()
    graph.replay()
    assert torch.equal(out, first)
    k[:, :, 30] *= 1e10  # now a tile is wide
    graph.replay()
    assert torch.equal(out, f())
    assert rel(out[:, :, 1340:], reference(q, k, v, 1300, 2, 0)[:, :, 1340:]) <= 1e-5
    k[:, :, 30] /= 1e10
    graph.replay()
    assert torch.equal(out, f())
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    want = f()
    torch.cuda.synchronize()
    got = []
    for _ in range(4):
        for stream in (a, b):
            with torch.cuda.stream(stream):
                got.append(f())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


@pytest.mark.parametrize("d", [32, 64, 128])
@pytest.mark.parametrize("s,w", [(300, 100), (1400, 1300), (5000, 4500)])
@pytest.mark.parametrize("big", [1e4, 1e8, 1e12, 1e18])
def test_huge_scores_pick_one_key(d, s, w, big):
    # One key's score is far above the others of every row (its gap passes 100): the row is that key's
    # value, up to the tolerance. Rows that do not see it keep theirs.
    q, k, v = make(1, 1, 1, s, s, d, "plain", 27)
    q[..., 0] = q[..., 0].abs() + 1.0
    k[:, :, 40] = 0
    k[:, :, 40, 0] = big
    out = F.sliding_window_attention(q, k, v, w)
    seen = slice(40, 40 + w)
    assert rel(out[:, :, seen], v[:, :, 40:41].expand_as(out[:, :, seen]).double()) <= 1e-5
    ref = reference(q, k, v, w, 0, 0)
    rest = torch.cat([out[:, :, :40], out[:, :, 40 + w:]], 2)
    assert rel(rest, torch.cat([ref[:, :, :40], ref[:, :, 40 + w:]], 2)) <= 1e-5
    assert dc._lib.load().dc_device_status(1) == 0


@pytest.mark.parametrize("layout", ["plain", "odd"])
@pytest.mark.parametrize("d", [32, 64, 128, 200])
@pytest.mark.parametrize("case", [  # l, s, window, sinks, offset, valid keys per sequence
    (1, 1, 1, 0, None, None), (1, 1, 9, 4, None, None), (300, 300, 1, 0, None, None), (70, 300, 1, 0, None, None),
    (200, 100, 50, 0, 149, None), (150, 150, 40, 0, 0, (1, 1)), (150, 150, 150, 3, 0, (1, 0)), (300, 300, 1, 0, 0, (200, 60)),
    (129, 2, 1, 1, 0, (1, 1))])
def test_rows_of_one_key_have_no_score_gradient(case, d, layout):
    # A row's only key has the weight 1 whatever its score: dq and dk are exactly 0, dv is grad_out's sum.
    l, s, window, sinks, offset, valid = case
    q, k, v = (t.detach().requires_grad_() for t in make(2, 4, 2, l, s, d, layout, 28))
    mask = None
    if valid:
        mask = (torch.arange(s, device="cuda") < torch.tensor(valid, device="cuda")[:, None])[:, None, None]
    out = F.sliding_window_attention(q, k, v, window, sinks, attn_mask=mask, offset=offset, enable_gqa=True)
    go = torch.randn(out.shape, device="cuda")
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), go)
    refs = [t.detach().double().requires_grad_() for t in (q, k, v)]
    ref = reference(*refs, window, sinks, s - l if offset is None else offset, mask)
    rq, rk, rv = torch.autograd.grad(ref, refs, go.double())
    one = [(x == 0).all().item() for x in (rq, rk)]
    if case != (200, 100, 50, 0, 149, None):
        assert one == [True, True]
        assert (dq == 0).all() and (dk == 0).all()
    for a, r in ((out, ref), (dv, rv), (dq, rq), (dk, rk)):
        assert rel(a.detach(), r.detach()) <= 1e-5


def test_rows_of_one_key_beside_others():
    # Every third row sees one key, the others all; float and bool masks, both tensor-core head dims.
    for d in (64, 128):
        q, k, v = make(1, 2, 2, 260, 260, d, "bshd", 29)
        i, j = torch.arange(260, device="cuda")[:, None], torch.arange(260, device="cuda")
        mask = (i % 3 != 0) | (j == i)
        for m in (mask, torch.where(mask, 0.25, -math.inf)):
            _, grads = check(q, k, v, 100, 2, mask=m)
            assert (grads[0][:, :, ::3] == 0).all()
