"""The native entry points, under the names DenseCore's pyo3 module exports.

``_flash_attention`` and ``_flash_attention_backward`` keep the signatures of
src/lib.rs:609-638 and :640-683 (``(q, k, v, causal, scale=None, mask=None)`` and
``(grad_out, q, k, v, out, lse, causal, scale=None, mask=None)``), their ValueError /
RuntimeError behaviour, and their outputs: fresh tensors (out, lse) and (grad_q, grad_k,
grad_v). The tensors are CUDA ``torch.Tensor`` (torch is used for device memory and streams
only); the work runs in libdensecore_sdpa.so. ``mask`` may be any float32/bool tensor that
broadcasts to (B, H, L, S) -- for a bool mask True means "may attend" -- so DenseCore's
materialised (B, H, L, S) float mask is accepted as one case of it.
"""
from __future__ import annotations

import contextlib
import functools

import torch

from . import _lib
from .backends import precision_code


def _require_cuda(*ts):
    dev = None
    for t in ts:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError("flash attention takes torch.Tensor arguments")
        if not t.is_cuda:
            raise RuntimeError("densecore_b200 runs on CUDA tensors; got a tensor on " + str(t.device))
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise RuntimeError(f"flash attention tensors are on different devices ({dev}, {t.device})")
    return dev


def _scale_args(scale):
    return (0, 0.0) if scale is None else (1, float(scale))


def _flash_attention(q, k, v, causal, scale=None, mask=None, precision=None):
    """Forward: (out (B,H,L,Ev), lse (B,H,L)). src/lib.rs:609-638."""
    L = _lib.load()
    dev = _require_cuda(q, k, v, mask)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("flash attention takes (B, H, L, E) tensors")
    B, H, Lq = q.shape[:3]
    out = torch.empty((B, H, Lq, v.shape[3]), device=dev, dtype=torch.float32)
    lse = torch.empty((B, H, Lq), device=dev, dtype=torch.float32)
    prec = precision_code() if precision is None else precision
    has, sc = _scale_args(scale)
    with torch.cuda.device(dev):
        vq, vk, vv, vm, vo, vl = (_lib.view(t) for t in (q, k, v, mask, out, lse))
        path = L.dc_sdpa_fwd_path(_lib.ref(vq), _lib.ref(vk), _lib.ref(vv), _lib.ref(vm), int(bool(causal)), prec)
        if path == 2:
            splits = L.dc_sdpa_decode_default_splits(B, H, k.shape[2])
            ws = torch.empty(max(L.dc_sdpa_decode_workspace_size(B, H, v.shape[3], splits), 1),
                             dtype=torch.uint8, device=dev)
            st = L.dc_sdpa_decode(_lib.ref(vq), _lib.ref(vk), _lib.ref(vv), _lib.ref(vm), has, sc, splits,
                                  _lib.ref(vo), _lib.ref(vl), ws.data_ptr(), ws.numel(), _lib.stream_of(q))
        else:
            st = L.dc_sdpa_fwd(_lib.ref(vq), _lib.ref(vk), _lib.ref(vv), _lib.ref(vm), int(bool(causal)), has, sc,
                               prec, _lib.ref(vo), _lib.ref(vl), _lib.stream_of(q))
    _lib.check(st, "flash attention forward failed")
    return out, lse


def _flash_attention_backward(grad_out, q, k, v, out, lse, causal, scale=None, mask=None, precision=None):
    """Backward: (grad_q, grad_k, grad_v). src/lib.rs:640-683."""
    L = _lib.load()
    dev = _require_cuda(grad_out, q, k, v, out, lse, mask)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("flash attention takes (B, H, L, E) tensors")
    gq = torch.empty(q.shape, device=dev, dtype=torch.float32)
    gk = torch.empty(k.shape, device=dev, dtype=torch.float32)
    gv = torch.empty(v.shape, device=dev, dtype=torch.float32)
    prec = precision_code() if precision is None else precision
    has, sc = _scale_args(scale)
    with torch.cuda.device(dev):
        nbytes = L.dc_sdpa_bwd_workspace_size(q.shape[0], q.shape[1], q.shape[2])
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)
        views = [_lib.view(t) for t in (grad_out, q, k, v, out, lse, mask, gq, gk, gv)]
        st = L.dc_sdpa_bwd(*[_lib.ref(x) for x in views[:7]], int(bool(causal)), has, sc, prec,
                           *[_lib.ref(x) for x in views[7:]], ws.data_ptr(), ws.numel(), _lib.stream_of(q))
    _lib.check(st, "flash attention backward failed")
    return gq, gk, gv


def _flash_attention_dropout(q, k, v, causal, scale, mask, keep, keep_scale, precision=None):
    """Forward with dropout on the weights (dc_sdpa_fwd_dropout): (out, lse). ``keep`` holds
    the packed keep bits of the (B, H, L, S) weights, ``keep_scale`` = float32(1/(1-p))."""
    L = _lib.load()
    dev = _require_cuda(q, k, v, mask, keep)
    if q.dim() != 4 or k.dim() != 4 or v.dim() != 4:
        raise ValueError("flash attention takes (B, H, L, E) tensors")
    B, H, Lq = q.shape[:3]
    out = torch.empty((B, H, Lq, v.shape[3]), device=dev, dtype=torch.float32)
    lse = torch.empty((B, H, Lq), device=dev, dtype=torch.float32)
    prec = precision_code() if precision is None else precision
    has, sc = _scale_args(scale)
    with torch.cuda.device(dev):
        vs = [_lib.view(t) for t in (q, k, v, mask, out, lse)]
        st = L.dc_sdpa_fwd_dropout(*[_lib.ref(x) for x in vs[:4]], int(bool(causal)), has, sc, prec, keep.data_ptr(),
                                   float(keep_scale), _lib.ref(vs[4]), _lib.ref(vs[5]), _lib.stream_of(q))
    _lib.check(st, "flash attention forward failed")
    return out, lse


def _flash_attention_dropout_backward(grad_out, q, k, v, out, lse, causal, scale, mask, keep, keep_scale,
                                      precision=None):
    """Backward of :func:`_flash_attention_dropout` (dc_sdpa_bwd_dropout): (grad_q, grad_k, grad_v)."""
    L = _lib.load()
    dev = _require_cuda(grad_out, q, k, v, out, lse, mask, keep)
    gq = torch.empty(q.shape, device=dev, dtype=torch.float32)
    gk = torch.empty(k.shape, device=dev, dtype=torch.float32)
    gv = torch.empty(v.shape, device=dev, dtype=torch.float32)
    prec = precision_code() if precision is None else precision
    has, sc = _scale_args(scale)
    with torch.cuda.device(dev):
        nbytes = L.dc_sdpa_bwd_workspace_size(q.shape[0], q.shape[1], q.shape[2])
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=dev)
        views = [_lib.view(t) for t in (grad_out, q, k, v, out, lse, mask, gq, gk, gv)]
        st = L.dc_sdpa_bwd_dropout(*[_lib.ref(x) for x in views[:7]], int(bool(causal)), has, sc, prec,
                                   keep.data_ptr(), float(keep_scale), *[_lib.ref(x) for x in views[7:]],
                                   ws.data_ptr(), ws.numel(), _lib.stream_of(q))
    _lib.check(st, "flash attention backward failed")
    return gq, gk, gv


def _decode(q, k, v, scale=None, mask=None, num_splits=0, workspace=None):
    """Split-KV decode for q_len == 1 (dc_sdpa_decode): (out, lse)."""
    L = _lib.load()
    dev = _require_cuda(q, k, v, mask)
    B, H, Lq = q.shape[:3]
    out = torch.empty((B, H, Lq, v.shape[3]), device=dev, dtype=torch.float32)
    lse = torch.empty((B, H, Lq), device=dev, dtype=torch.float32)
    has, sc = _scale_args(scale)
    with torch.cuda.device(dev):
        splits = num_splits if num_splits > 0 else L.dc_sdpa_decode_default_splits(B, H, k.shape[2])
        need = L.dc_sdpa_decode_workspace_size(B, H, v.shape[3], splits)
        ws = workspace if workspace is not None else torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
        vs = [_lib.view(t) for t in (q, k, v, mask, out, lse)]
        st = L.dc_sdpa_decode(*[_lib.ref(x) for x in vs[:4]], has, sc, splits, _lib.ref(vs[4]), _lib.ref(vs[5]),
                              ws.data_ptr(), ws.numel(), _lib.stream_of(q))
    _lib.check(st, "decode attention failed")
    return out, lse


def _attn_merge(out_acc, lse_acc, out_part, lse_part):
    """In-place logsumexp merge of (out_part, lse_part) into (out_acc, lse_acc)."""
    L = _lib.load()
    _require_cuda(out_acc, lse_acc, out_part, lse_part)
    with torch.cuda.device(out_acc.device):
        vs = [_lib.view(t) for t in (out_acc, lse_acc, out_part, lse_part)]
        st = L.dc_attn_merge(*[_lib.ref(x) for x in vs], _lib.stream_of(out_acc))
    _lib.check(st, "attention merge failed")
    return out_acc, lse_acc


def _ring_attention(q, k, v, comm_ptr, causal=True, scale=None, precision=None, workspace=None):
    """Ring attention forward of this rank's zig-zag shards over an NCCL communicator
    (dc_ring_sdpa_fwd): (out, lse) of the local query rows against the whole sequence."""
    L = _lib.load()
    dev = _require_cuda(q, k, v)
    B, H, Lq = q.shape[:3]
    out = torch.empty((B, H, Lq, v.shape[3]), device=dev, dtype=torch.float32)
    lse = torch.empty((B, H, Lq), device=dev, dtype=torch.float32)
    prec = precision_code() if precision is None else precision
    has, sc = _scale_args(scale)
    with torch.cuda.device(dev):
        need = L.dc_ring_sdpa_fwd_workspace_size(B, H, k.shape[1], Lq, q.shape[3])
        ws = workspace if workspace is not None else torch.empty(max(need, 1), dtype=torch.uint8, device=dev)
        vs = [_lib.view(t) for t in (q, k, v, out, lse)]
        st = L.dc_ring_sdpa_fwd(*[_lib.ref(x) for x in vs[:3]], int(bool(causal)), has, sc, prec, comm_ptr,
                                _lib.ref(vs[3]), _lib.ref(vs[4]), ws.data_ptr(), ws.numel(), _lib.stream_of(q))
    _lib.check(st, "ring attention failed")
    return out, lse


def _attn_probs(q, k, lse, causal, scale=None, mask=None, average_heads=True, keep=None, keep_scale=0.0):
    """softmax(scale q k^T + mask) from the forward's lse; (B,L,S) head mean or (B,H,L,S).
    With ``keep`` (packed dropout keep bits) each probability is times its dropout factor."""
    L = _lib.load()
    dev = _require_cuda(q, k, lse, mask, keep)
    B, H, Lq = q.shape[:3]
    S = k.shape[2]
    shape = (B, Lq, S) if average_heads else (B, H, Lq, S)
    probs = torch.empty(shape, device=dev, dtype=torch.float32)
    has, sc = _scale_args(scale)
    with torch.cuda.device(dev):
        vs = [_lib.view(t) for t in (q, k, lse, mask, probs)]
        if keep is None:
            st = L.dc_attn_probs(*[_lib.ref(x) for x in vs[:4]], int(bool(causal)), has, sc,
                                 int(bool(average_heads)), _lib.ref(vs[4]), _lib.stream_of(q))
        else:
            st = L.dc_attn_probs_dropout(*[_lib.ref(x) for x in vs[:4]], int(bool(causal)), has, sc, keep.data_ptr(),
                                         float(keep_scale), int(bool(average_heads)), _lib.ref(vs[4]),
                                         _lib.stream_of(q))
    _lib.check(st, "attention probabilities failed")
    return probs


def _fwd_path(q, k, v, mask=None, causal=False, precision=None):
    """0 = CUDA-core kernels, 1 = tcgen05 tensor cores, 2 = split-KV decode."""
    L = _lib.load()
    prec = precision_code() if precision is None else precision
    vs = [_lib.view(t) for t in (q, k, v, mask)]
    return L.dc_sdpa_fwd_path(*[_lib.ref(x) for x in vs], int(bool(causal)), prec)


_PROXY = torch._C._TorchDispatchModeKey.PROXY
_PRE_DISPATCH = torch._ops.mode_stack_state_for_pre_dispatch()
_mode_count, _is_tracing = torch._C._len_torch_dispatch_stack, torch._C._is_tracing


def _traced(what):
    """Whether torch.jit.trace is recording: of a call outside an autograd Function it would record the
    allocations alone, and the trace return them unwritten. make_fx records no Function either: refused."""
    if _mode_count() and torch._C._get_dispatch_mode(_PROXY) is not None or _PRE_DISPATCH.get(0) is not None:
        raise RuntimeError(f"{what} cannot be recorded by make_fx")
    return _is_tracing()


_SAME_DEVICE = contextlib.nullcontext()


def _on(dev):
    """The context in which ``dev`` is the current device."""
    return _SAME_DEVICE if torch._C._cuda_getDevice() == dev.index else torch.cuda.device(dev)


def _device_of(first, *rest):
    """:func:`_require_cuda` with one integer comparison a tensor while all is well."""
    index = first.get_device()
    if index >= 0:
        for t in rest:
            if t is not None and t.get_device() != index:
                break
        else:
            return first.device
    return _require_cuda(first, *rest)


def _refs(*ts):
    """The tensors as the C entry points take them (None stays None)."""
    return [_lib.packed(t) for t in ts]


def _stream(dev):
    return torch._C._cuda_getCurrentRawStream(dev.index)


# Scratch sizes depend on sizes (and the device's SM count) only; asking the library costs as much as a
# launch, which shows in single-token calls. `index`: the device's.
@functools.lru_cache(maxsize=1024)
def _window_scratch(index, *sizes):
    return _lib.load().dc_sdpa_window_fwd_workspace_size(*sizes)


@functools.lru_cache(maxsize=1024)
def _cache4_scratch(index, *sizes):
    return _lib.load().dc_cache4_attention_workspace_size(*sizes)


def _decode_buffers(like, rows_shape, scratch, need_lse):
    """(logsumexp or None, its packed view, scratch pointer, the tensor that holds the scratch): a
    logsumexp that nobody asked for lies behind the scratch, in one allocation."""
    b, h = rows_shape
    if need_lse:
        lse = torch.empty((b, h, 1), device=like.device, dtype=torch.float32)
        hold = torch.empty(scratch, dtype=torch.uint8, device=like.device) if scratch else None
        return lse, _lib.packed(lse), hold.data_ptr() if scratch else None, hold
    at = (scratch + 15) // 16 * 16
    hold = torch.empty(at + 4 * b * h, dtype=torch.uint8, device=like.device)
    ptr = hold.data_ptr()
    return None, _lib._PACK[3](ptr + at, _lib.DC_F32, 3, b, h, 1, h, 1, 1), ptr if scratch else None, hold


def _sliding_window(q, k, v, window, sinks, offset, scale=None, mask=None, lengths=None, precision=None, need_lse=True):
    """Forward through a sliding window (dc_sdpa_window_fwd): (out, lse); one query row without
    ``need_lse``: (out, None)."""
    L = _lib.load()
    dev = _device_of(q, k, v, mask, lengths)
    B, H, Lq, E = q.shape
    Hkv, S, Ev = k.shape[1], k.shape[2], v.shape[3]
    if type(B) is not int:  # in a trace they come as tensors
        B, H, Lq, E, Hkv, S, Ev = map(int, (B, H, Lq, E, Hkv, S, Ev))
    out = torch.empty_like(q) if E == Ev else torch.empty((B, H, Lq, Ev), device=dev, dtype=torch.float32)
    prec = precision_code() if precision is None else precision
    has, sc = _scale_args(scale)
    with _on(dev):
        if Lq == 1:
            need = _window_scratch(dev.index, B, H, Hkv, Lq, S, E, window, sinks) if Hkv and H % Hkv == 0 else 0
            lse, lse_ref, ptr, _hold = _decode_buffers(q, (B, H), need, need_lse)
        else:
            need, ptr = 0, None
            lse = torch.empty((B, H, Lq), device=dev, dtype=torch.float32)
            lse_ref = _lib.packed(lse)
        r = _refs(q, k, v, mask, lengths, out)
        st = L.dc_sdpa_window_fwd(*r[:4], window, sinks, offset, r[4], has, sc, prec, r[5], lse_ref, ptr, need,
                                  _stream(dev))
    _lib.check(st, "sliding window attention failed")
    return out, lse


def _sliding_window_backward(grad_out, q, k, v, out, lse, window, sinks, offset, scale=None, mask=None, precision=None):
    """Backward of :func:`_sliding_window` (dc_sdpa_window_bwd): (grad_q, grad_k, grad_v)."""
    L = _lib.load()
    dev = _device_of(grad_out, q, k, v, out, lse, mask)
    gq = torch.empty(q.shape, device=dev, dtype=torch.float32)
    gk = torch.empty(k.shape, device=dev, dtype=torch.float32)
    gv = torch.empty(v.shape, device=dev, dtype=torch.float32)
    prec = precision_code() if precision is None else precision
    has, sc = _scale_args(scale)
    with _on(dev):
        nbytes = max(L.dc_sdpa_bwd_workspace_size(q.shape[0], q.shape[1], q.shape[2]), 1)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        r = _refs(grad_out, q, k, v, out, lse, mask, gq, gk, gv)
        st = L.dc_sdpa_window_bwd(*r[:7], window, sinks, offset, has, sc, prec, *r[7:], ws.data_ptr(), nbytes,
                                  _stream(dev))
    _lib.check(st, "sliding window attention backward failed")
    return gq, gk, gv


def _rotary(q, k, positions, inv_freq, interleaved, amplitude, inverse=False):
    """Rotary positions of (B, H, L, D) q and k (or None), or the inverse turn (dc_rotary)."""
    L = _lib.load()
    dev = _device_of(q, k, positions, inv_freq)
    yq = torch.empty_like(q)
    yk = None if k is None else torch.empty_like(k)
    with _on(dev):
        r = _refs(q, k, positions, inv_freq, yq, yk)
        st = L.dc_rotary(*r[:4], int(interleaved), amplitude, int(inverse), r[4], r[5], _stream(dev))
    _lib.check(st, "rotary positions failed")
    return yq, yk


def _qk_norm_rotary(q, k, wq, wk, positions, inv_freq, eps, interleaved, amplitude):
    """Rotary positions of each head's row over its root mean square (dc_qk_norm_rotary)."""
    L = _lib.load()
    dev = _device_of(q, k, wq, wk, positions, inv_freq)
    yq = torch.empty_like(q)
    yk = None if k is None else torch.empty_like(k)
    with _on(dev):
        r = _refs(q, k, wq, wk, positions, inv_freq, yq, yk)
        st = L.dc_qk_norm_rotary(*r[:6], eps, int(interleaved), amplitude, r[6], r[7], _stream(dev))
    _lib.check(st, "normed rotary positions failed")
    return yq, yk


def _qk_norm_rotary_backward(gyq, gyk, q, k, wq, wk, positions, inv_freq, eps, interleaved, amplitude,
                             weight_grads=(True, True)):
    """Backward of :func:`_qk_norm_rotary`: (grad_q, grad_k, grad_wq, grad_wk); a weight's gradient is
    None where there is no weight or ``weight_grads`` says it is not needed."""
    L = _lib.load()
    dev = _device_of(gyq, gyk, q, k, wq, wk, positions, inv_freq)
    gq = torch.empty_like(q)
    gk = None if k is None else torch.empty_like(k)
    gws = [torch.empty_like(w) if w is not None and need else None for w, need in zip((wq, wk), weight_grads)]
    with _on(dev):
        nbytes = L.dc_qk_norm_rotary_bwd_workspace_size(q.shape[3])
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
        r = _refs(gyq, gyk, q, k, wq, wk, positions, inv_freq, gq, gk, *gws)
        st = L.dc_qk_norm_rotary_bwd(*r[:8], eps, int(interleaved), amplitude, *r[8:], ws.data_ptr(), nbytes,
                                     _stream(dev))
    _lib.check(st, "normed rotary positions backward failed")
    return gq, gk, gws[0], gws[1]


def _cache4_append(desc, key, value, page_table, start, end=None):
    """Tokens into a 4-bit cache (dc_cache4_append); ``desc`` is a ``_lib.DcCache4``."""
    L = _lib.load()
    dev = _device_of(key, value, page_table, start, end)
    with _on(dev):
        st = L.dc_cache4_append(_lib.ref(desc), *_refs(key, value, page_table, start, end), _stream(dev))
    _lib.check(st, "cache append failed")


def _cache4_read(desc, page_table, lengths, max_length):
    """The first max_length positions of each sequence (dc_cache4_read): (key, value) in float32."""
    L = _lib.load()
    dev = _device_of(page_table, lengths)
    shape = (page_table.shape[0], desc.kv_heads, max_length, desc.head_dim)
    key = torch.empty(shape, device=dev, dtype=torch.float32)
    value = torch.empty(shape, device=dev, dtype=torch.float32)
    with _on(dev):
        st = L.dc_cache4_read(_lib.ref(desc), *_refs(page_table, lengths, key, value), _stream(dev))
    _lib.check(st, "cache read failed")
    return key, value


def _cache4_attention(desc, q, page_table, lengths, window=0, sinks=0, scale=None, need_lse=True):
    """One token per sequence over a 4-bit cache (dc_cache4_attention): (out, lse), or (out, None)
    without ``need_lse``."""
    L = _lib.load()
    dev = _device_of(q, page_table, lengths)
    B, H = q.shape[:2]
    out = torch.empty_like(q)
    has, sc = _scale_args(scale)
    with _on(dev):
        kv = desc.kv_heads
        need = _cache4_scratch(dev.index, B, H, kv, desc.head_dim, page_table.shape[1] * desc.page_size, window, sinks,
                               _lib._DTYPES[q.dtype]) if H and H % kv == 0 else 0
        lse, lse_ref, ptr, _hold = _decode_buffers(q, (B, H), need, need_lse)
        q_, table_, lengths_, out_ = _refs(q, page_table, lengths, out)
        st = L.dc_cache4_attention(_lib.ref(desc), q_, table_, lengths_, window, sinks, has, sc, out_, lse_ref, ptr, need,
                                   _stream(dev))
    _lib.check(st, "cache attention failed")
    return out, lse
