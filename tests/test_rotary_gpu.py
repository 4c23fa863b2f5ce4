"""Rotary positions and normed queries and keys against the formulas in 64 bits.

Tolerances. The angle is a float32 fraction of a turn (off by 2^-25 turns, 1.9e-7 rad), its sine and
cosine are off by 2 units in the last place at most (2.4e-7), the amplitude, the two products and
their sum round once each (4 * 2^-24): below 1e-6 of (|a| + |b|) * amplitude for a pair. The norm adds
the sum of up to 256 squares over chains of at most 16 + 5 terms, halved by the square root (11 *
2^-24), and five roundings: 2e-6 together, so 3e-6 in all. An output in 16 bits is off by half a step
more."""
import math

import pytest
import torch

import densecore_b200 as dc
from densecore_b200 import functional as F

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def turn(x, angle, amplitude, interleaved, magnitude=False):
    """The rotation in 64 bits; with magnitude, the sum of the absolute terms of each channel."""
    r = angle.shape[-1]
    y = x.clone()
    a, b = (x[..., 0:2 * r:2], x[..., 1:2 * r:2]) if interleaved else (x[..., :r], x[..., r:2 * r])
    if magnitude:
        a = b = (a.abs() + b.abs()) * amplitude
        y = x.abs()
    else:
        c, s = angle.cos() * amplitude, angle.sin() * amplitude
        a, b = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:2 * r:2], y[..., 1:2 * r:2] = a, b
    else:
        y[..., :r], y[..., r:2 * r] = a, b
    return y


def angles(positions, freq, b):
    p = positions if positions.dim() == 2 else positions[None]
    return p.double().expand(b, -1)[:, None, :, None] * freq


def close(got, ref, size, rel):
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != torch.float32 else 0.0
    tol = rel * size + half * (ref.abs() + rel * size) + torch.finfo(got.dtype).tiny
    bad = (got.double() - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got.double() - ref).abs() / tol).max()))


def make(b, h, kv, l, d, dtype, layout, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if layout == "fused":
        x = torch.randn(b, l, (h + 2 * kv) * d, generator=g, device="cuda").to(dtype)
        q = x[..., :h * d].view(b, l, h, d).transpose(1, 2)
        k = x[..., h * d:(h + kv) * d].view(b, l, kv, d).transpose(1, 2)
    elif layout == "odd":  # rows off every 16-byte boundary, elements two apart
        q = torch.randn(b, h, l, 2 * d + 1, generator=g, device="cuda").to(dtype)[..., 1::2]
        k = torch.randn(b, kv, l, 2 * d + 1, generator=g, device="cuda").to(dtype)[..., 1::2]
    else:
        q, k = (torch.randn(b, n, l, d, generator=g, device="cuda").to(dtype) for n in (h, kv))
    return q, k


SHAPES = [  # b, h, kv, l, d, rotated
    (1, 1, 1, 1, 2, 2), (2, 3, 1, 5, 64, 64), (3, 32, 8, 1, 128, 128), (2, 12, 12, 33, 64, 32), (1, 8, 2, 130, 80, 80),
    (1, 5, 5, 7, 96, 16), (2, 4, 2, 9, 256, 256), (1, 2, 1, 3, 254, 10), (1, 40, 8, 300, 128, 64), (2, 7, 3, 4, 6, 4)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["plain", "fused", "odd"])
@pytest.mark.parametrize("shape", SHAPES)
def test_rotary_forward_and_backward(shape, layout, interleaved, dtype):
    b, h, kv, l, d, rot = shape
    q, k = make(b, h, kv, l, d, dtype, layout)
    freq, amp = F.rotary_frequencies(rot, device="cuda")
    amp = 1.25
    pos = torch.arange(l, device="cuda") + 100 * torch.arange(b, device="cuda")[:, None]
    ang = angles(pos, freq, b)
    qg, kg = q.detach().requires_grad_(), k.detach().requires_grad_()
    yq, yk = F.rotary_embedding(qg, kg, pos, freq, interleaved=interleaved, amplitude=amp)
    gq, gk = (torch.randn_like(y) for y in (yq, yk))
    dq, dk = torch.autograd.grad((yq, yk), (qg, kg), (gq, gk))
    for x, y, g, dx in ((q, yq, gq, dq), (k, yk, gk, dk)):
        assert y.shape == x.shape and y.dtype == dtype
        xd, gd = x.double(), g.double()
        close(y, turn(xd, ang, amp, interleaved), turn(xd, ang, amp, interleaved, True), 1e-6)
        close(dx, turn(gd, -ang, amp, interleaved), turn(gd, ang, amp, interleaved, True), 1e-6)
        if rot < d:
            assert torch.equal(y[..., rot:], x[..., rot:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("layout", ["plain", "fused", "odd"])
@pytest.mark.parametrize("shape", SHAPES)
def test_norm_rotary_forward_and_backward(shape, layout, interleaved, dtype):
    b, h, kv, l, d, rot = shape
    q, k = make(b, h, kv, l, d, dtype, layout, 1)
    freq, amp = F.rotary_frequencies(rot, device="cuda")
    pos = torch.arange(l, device="cuda", dtype=torch.int32) * 3
    ang = angles(pos, freq, b)
    g = torch.Generator(device="cuda").manual_seed(5)
    wq = (1 + 0.3 * torch.randn(d, generator=g, device="cuda")).to(dtype)
    wk = 1 + 0.3 * torch.randn(d, generator=g, device="cuda")  # float32 beside 16-bit rows too
    leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
    eps = 1e-5
    yq, yk = F.qk_norm_rotary(*leaves, pos, freq, eps=eps, interleaved=interleaved, amplitude=amp)
    gq, gk = (torch.randn_like(y) for y in (yq, yk))
    dq, dk, dwq, dwk = torch.autograd.grad((yq, yk), leaves, (gq, gk))
    for x, w, y, gy, dx, dw in ((q, wq, yq, gq, dq, dwq), (k, wk, yk, gk, dk, dwk)):
        xd, wd, gd = x.double(), w.double(), gy.double()
        r = 1 / (xd.square().mean(-1, keepdim=True) + eps).sqrt()
        n = xd * r
        close(y, turn(n * wd, ang, amp, interleaved), turn(n * wd, ang, amp, interleaved, True), 3e-6)
        u, us = turn(gd, -ang, amp, interleaved), turn(gd, ang, amp, interleaved, True)
        gn, gns = u * wd, us * wd.abs()
        ref = r * (gn - n * (gn * n).mean(-1, keepdim=True))
        # the mean of D products sums like the squares: 3e-6 of its absolute terms, as gn and n are
        close(dx, ref, r * (gns + n.abs() * (gns * n.abs()).mean(-1, keepdim=True)), 6e-6)
        rows = b * x.shape[1] * l
        # a sum of `rows` terms in any order: (rows - 1) roundings of at most the absolute sum
        close(dw, (u * n).sum((0, 1, 2)), (us * n.abs()).sum((0, 1, 2)), 3e-6 + rows * 2.0 ** -24)


def test_gradients_agree_with_differences():
    # L = sum(y * c) is smooth; the central difference over 2 h has error h^2/6 L''' + 2^-24 |L| / h.
    torch.manual_seed(0)
    q = torch.randn(1, 2, 3, 8, device="cuda")
    w = 1 + 0.2 * torch.randn(8, device="cuda")
    c = torch.randn(1, 2, 3, 8, device="cuda")
    freq, _ = F.rotary_frequencies(8, device="cuda")
    pos = torch.arange(3, device="cuda")

    def loss(q, w):
        return (F.qk_norm_rotary(q, None, w, None, pos, freq)[0].double() * c).sum()

    ql, wl = q.clone().requires_grad_(), w.clone().requires_grad_()
    loss(ql, wl).backward()
    h = 1.0 / 64
    for leaf, base, args in ((ql, q, 0), (wl, w, 1)):
        for i in (0, 3, 7):
            d = torch.zeros_like(base).view(-1)
            d[i] = h
            d = d.view_as(base)
            up, down = ((loss(q + s * d, w) if args == 0 else loss(q, w + s * d)) for s in (1, -1))
            assert abs(float((up - down) / (2 * h)) - float(leaf.grad.view(-1)[i])) < 2e-3


def test_far_positions_and_scaled_frequencies():
    freq, amp = F.rotary_frequencies(128, scaling="yarn", factor=4.0, original_length=8192, device="cuda")
    q = torch.randn(1, 2, 4, 128, device="cuda")
    pos = torch.tensor([0, 10 ** 6 + 7, 2 ** 31 + 5, -3], device="cuda")
    y, none = F.rotary_embedding(q, None, pos, freq, amplitude=amp)
    assert none is None
    # positions * freq in 64 bits is off by 2^-53 of up to 2^31 rad: below 5e-7 rad
    close(y, turn(q.double(), angles(pos, freq, 1), amp, False), turn(q.double(), angles(pos, freq, 1), amp, False, True), 2e-6)


def test_rank_three_broadcast_gradients_and_unused_outputs():
    freq, _ = F.rotary_frequencies(16, device="cuda")
    pos = torch.arange(5, device="cuda")
    q = torch.randn(2, 5, 16, device="cuda", requires_grad=True)
    k = torch.randn(2, 5, 16, device="cuda", requires_grad=True)
    y, _ = F.rotary_embedding(q, k, pos, freq)
    y.sum().backward()  # an expanded gradient; the key's output is not used
    ref = turn(torch.ones(2, 1, 5, 16, device="cuda").double(), -angles(pos, freq, 2), 1.0, False)[:, 0]
    close(q.grad, ref, torch.full_like(ref, 2.0), 1e-6)
    assert torch.equal(k.grad, torch.zeros_like(k))
    w = torch.ones(16, device="cuda")
    y, _ = F.qk_norm_rotary(q, k, w, None, pos, freq)
    q.grad = None
    y.sum().backward()
    assert q.grad is not None and torch.isfinite(q.grad).all()


def test_empty_calls():
    freq, _ = F.rotary_frequencies(16, device="cuda")
    for b, h, l in ((0, 2, 3), (2, 0, 3), (2, 2, 0)):
        q = torch.randn(b, h, l, 16, device="cuda", requires_grad=True)
        w = torch.ones(16, device="cuda", requires_grad=True)
        pos = torch.arange(l, device="cuda")
        y, _ = F.rotary_embedding(q, None, pos, freq)
        assert y.shape == q.shape
        y, _ = F.qk_norm_rotary(q, None, w, None, pos, freq)
        y.sum().backward()
        assert torch.equal(w.grad, torch.zeros_like(w)) and q.grad.shape == q.shape


def test_weight_gradients_repeat_bit_for_bit_over_many_blocks():
    b, h, kv, l, d = 4, 32, 8, 1000, 128
    q, k = make(b, h, kv, l, d, torch.bfloat16, "fused", 3)
    freq, _ = F.rotary_frequencies(d, device="cuda")
    pos = torch.arange(l, device="cuda")
    w = torch.ones(d, device="cuda")
    gq, gk = torch.randn(b, h, l, d, device="cuda").bfloat16(), torch.randn(b, kv, l, d, device="cuda").bfloat16()
    runs = []
    for _ in range(3):
        leaves = [t.detach().requires_grad_() for t in (q, k, w, w)]
        runs.append(torch.autograd.grad(F.qk_norm_rotary(*leaves, pos, freq), leaves, (gq, gk)))
    for other in runs[1:]:
        assert all(torch.equal(x, y) for x, y in zip(runs[0], other))
    xd, gd = q.double(), gq.double()
    n = xd / (xd.square().mean(-1, keepdim=True) + 1e-6).sqrt()
    ang = angles(pos, freq, b)
    u, us = turn(gd, -ang, 1.0, False), turn(gd, ang, 1.0, False, True)
    # 128,000 rows over 592 blocks of 8 warps of 4 lane groups: chains of at most 40 rows a lane, then
    # 2 + 8 + 19 + 32 terms: 101 roundings
    close(runs[0][2], (u * n).sum((0, 1, 2)), (us * n.abs()).sum((0, 1, 2)), 3e-6 + 101 * 2.0 ** -24)


def test_in_place_and_streams():
    from densecore_b200 import _lib, _native
    q = torch.randn(2, 4, 6, 64, device="cuda")
    freq, _ = F.rotary_frequencies(64, device="cuda")
    pos = torch.arange(6, device="cuda")
    ref, _ = F.rotary_embedding(q, None, pos, freq)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        L = _lib.load()
        r = _native._refs(q, pos, freq)
        _lib.check(L.dc_rotary(r[0], None, r[1], r[2], 0, 1.0, 0, r[0], None, torch.cuda.current_stream().cuda_stream), "rotary")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(q, ref)
    assert dc._lib.load().dc_device_status(0) == 0
    assert math.isfinite(float(q.sum()))


def test_nothing_to_turn_and_infinities_that_pass_through():
    q = torch.randn(1, 2, 3, 64, device="cuda")
    q[0, 0, 0, 40] = math.inf
    pos = torch.arange(3, device="cuda")
    none = torch.empty(0, dtype=torch.float64, device="cuda")
    assert torch.equal(F.rotary_embedding(q, None, pos, none, amplitude=2.0)[0], q)
    freq, _ = F.rotary_frequencies(32, device="cuda")
    y, _ = F.rotary_embedding(q, None, pos, freq)
    assert torch.equal(y[..., 32:], q[..., 32:])


def test_more_than_two_to_the_31_elements():
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs memory")
    l, h, d = 560_000, 32, 128  # 2.3e9 elements
    x = torch.empty(1, l, h, d, dtype=torch.bfloat16, device="cuda").normal_()
    freq, _ = F.rotary_frequencies(d, device="cuda")
    pos = torch.arange(l, device="cuda")
    y, _ = F.rotary_embedding(x.transpose(1, 2), None, pos, freq)
    tail, _ = F.rotary_embedding(x[:, -5:].transpose(1, 2).contiguous(), None, pos[-5:], freq)
    assert torch.equal(y[:, :, -5:], tail)
    head, _ = F.rotary_embedding(x[:, :5].transpose(1, 2).contiguous(), None, pos[:5], freq)
    assert torch.equal(y[:, :, :5], head)
