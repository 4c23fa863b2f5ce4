"""Traces, tangents and gradients of the operators around attention, with stand-ins for the device calls
that copy their input on the CPU behind torch's back, as the kernels write their outputs."""
import ctypes

import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

import densecore_b200 as dc
from densecore_b200 import _native
from densecore_b200 import functional as F

POS = torch.arange(3)
FREQ, _ = F.rotary_frequencies(8)


def copied(t):
    """A copy that no tracer, tangent or graph sees."""
    if t is None:
        return None
    out = torch.empty_like(t)
    ctypes.memmove(out.data_ptr(), t.data_ptr(), t.numel() * t.element_size())
    return out


@pytest.fixture(autouse=True)
def on_the_cpu(monkeypatch):
    def window(q, k, v, window, sinks, offset, scale=None, mask=None, lengths=None, precision=None, need_lse=True):
        assert all(type(x) is int for x in (window, sinks, offset))
        assert lengths is not None or offset == k.shape[2] - q.shape[2]
        return copied(q), torch.zeros(q.shape[:3])

    monkeypatch.setattr(_native, "_sliding_window", window)
    monkeypatch.setattr(_native, "_rotary", lambda q, k, *a, **kw: (copied(q), copied(k)))
    monkeypatch.setattr(_native, "_qk_norm_rotary", lambda q, k, *a, **kw: (copied(q), copied(k)))
    monkeypatch.setattr(_native, "_cache4_attention", lambda desc, q, *a: (copied(q), None))
    monkeypatch.setattr(_native, "_cache4_read", lambda *a: (torch.empty(1), torch.empty(1)))
    monkeypatch.setattr(_native, "_cache4_append", lambda *a: None)


CALLS = {
    "rotary": lambda q: F.rotary_embedding(q, None, POS, FREQ)[0],
    "rotary of keys": lambda q: F.rotary_embedding(q + 1, q, POS, FREQ)[1],
    "norm": lambda q: F.qk_norm_rotary(q, None, torch.ones(8), None, POS, FREQ)[0],
    "norm of rank three": lambda q: F.qk_norm_rotary(q[0], q[0], None, None, POS, FREQ)[1][None],
    "window": lambda q: F.sliding_window_attention(q, q, q, 4),
    "window of few rows": lambda q: F.sliding_window_attention(q, torch.cat([q, q], 2), torch.cat([q, q], 2), 4),
    "masked window": lambda q: F.sliding_window_attention(q, q, q, 4, attn_mask=torch.ones(3, 3, dtype=torch.bool)),
}
LENGTHS = torch.ones(1, dtype=torch.int32)


def trace(call, q):
    return torch.jit.trace(call, (q,), check_trace=False)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_a_trace_keeps_the_call(name, grad):
    q, other = torch.randn(1, 2, 3, 8), torch.randn(1, 2, 3, 8)
    traced = trace(CALLS[name], q.requires_grad_(grad))
    assert torch.equal(traced(other), other)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_a_trace_takes_other_lengths():
    # The queries of a window are the last keys at every length, not at the traced one.
    traced = torch.jit.trace(lambda q, k: F.sliding_window_attention(q, k, k, 4), (torch.randn(1, 2, 3, 8), torch.randn(1, 2, 5, 8)),
                             check_trace=False)
    q, k = torch.randn(1, 2, 6, 8), torch.randn(1, 2, 11, 8)
    assert torch.equal(traced(q, k), q)
    one = torch.randn(1, 2, 1, 8)
    traced = torch.jit.trace(lambda q, k, n: F.sliding_window_attention(q, k, k, 4, lengths=n), (one, k, LENGTHS), check_trace=False)
    assert torch.equal(traced(2 * one, k, LENGTHS), 2 * one)


@pytest.mark.parametrize("mode", [dict(), dict(tracing_mode="fake"), dict(pre_dispatch=True)])
@pytest.mark.parametrize("name", CALLS)
def test_make_fx_is_refused(name, mode):
    with pytest.raises(RuntimeError, match="make_fx"):
        make_fx(CALLS[name], **mode)(torch.randn(1, 2, 3, 8))
    assert CALLS[name](torch.ones(1, 2, 3, 8)).shape == (1, 2, 3, 8)


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_a_cache_is_not_traced():
    cache = dc.KVCache4(2, 2, 64, page_size=16, device="cpu")
    table, k, q = torch.zeros(1, 1, dtype=torch.int32), torch.randn(1, 2, 1, 64), torch.randn(1, 4, 1, 64)
    for call in (lambda x: cache.attention(x, table, LENGTHS), lambda x: cache.append(k, k, table, LENGTHS),
                 lambda x: cache.read(table, LENGTHS, 1)):
        with pytest.raises(RuntimeError, match="traced"):
            trace(call, q)
        with pytest.raises(RuntimeError, match="make_fx"):
            make_fx(call)(q)
        call(q)


@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad])
@pytest.mark.parametrize("name", CALLS)
def test_tangents_are_refused_not_dropped(name, mode):
    q = torch.randn(1, 2, 3, 8)
    with mode(), forward_ad.dual_level():
        assert torch.equal(CALLS[name](q), q)  # no tangent, no refusal
        with pytest.raises(NotImplementedError, match="jvp"):
            CALLS[name](forward_ad.make_dual(q, torch.ones_like(q)))
    with pytest.raises(RuntimeError, match="functorch"):
        torch.func.jvp(CALLS[name], (q,), (q,))


def test_tangents_of_other_inputs_are_refused():
    q, k, w = torch.randn(1, 2, 1, 8), torch.randn(1, 2, 4, 8), torch.ones(8)
    at = torch.arange(1)
    calls = {
        "key": lambda d: F.sliding_window_attention(q, d(k), k, 4), "value": lambda d: F.sliding_window_attention(q, k, d(k), 4),
        "value of padded keys": lambda d: F.sliding_window_attention(q, k, d(k), 4, lengths=LENGTHS),
        "mask": lambda d: F.sliding_window_attention(q, k, k, 4, attn_mask=d(torch.zeros(1, 4))),
        "weight": lambda d: F.qk_norm_rotary(q, None, d(w), None, at, FREQ),
        "frequencies": lambda d: F.rotary_embedding(q, None, at, d(FREQ)),
    }
    for name, call in calls.items():
        call(lambda t: t)
        with forward_ad.dual_level():
            call(lambda t: t)
            with pytest.raises(NotImplementedError, match="jvp"):
                call(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))
    cache = dc.KVCache4(2, 2, 64, page_size=16, device="cpu")
    table, one = torch.zeros(1, 1, dtype=torch.int32), torch.randn(1, 4, 1, 64)
    with forward_ad.dual_level():
        assert torch.equal(cache.attention(one, table, LENGTHS), one)
        with pytest.raises(NotImplementedError, match="gradient"):
            cache.attention(forward_ad.make_dual(one, one), table, LENGTHS)


def test_frequencies_get_no_gradient():
    q, freq = torch.randn(1, 2, 3, 8), FREQ.clone().requires_grad_()
    for call in (lambda: F.rotary_embedding(q, None, POS, freq), lambda: F.qk_norm_rotary(q, q, None, None, POS, freq)):
        with pytest.raises(NotImplementedError, match="frequencies"):
            call()
        with torch.no_grad():
            assert torch.equal(call()[0], q)
