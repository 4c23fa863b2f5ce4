"""Refusals of the operators around attention: raised before any device work, so they run on the CPU."""
import ctypes
import math

import pytest
import torch

import densecore_b200 as dc
from densecore_b200 import _lib
from densecore_b200 import functional as F


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def test_sliding_window_refusals():
    q, k = t(1, 4, 3, 8), t(1, 2, 5, 8)
    call = F.sliding_window_attention
    with pytest.raises(TypeError, match="Tensor"):
        call(q.numpy(), k, k, 4)
    with pytest.raises(ValueError, match="rank"):
        call(q, k[0], k, 4)
    with pytest.raises(ValueError, match="shapes"):
        call(q, k, k, 4)  # grouped heads need enable_gqa
    with pytest.raises(ValueError, match="shapes"):
        call(t(1, 3, 3, 8), k, k, 4, enable_gqa=True)
    with pytest.raises(ValueError, match="shapes"):
        call(q, k, t(1, 2, 4, 8), 4, enable_gqa=True)
    ok = dict(enable_gqa=True)
    for window in (0, -3, 1 << 70):
        with pytest.raises(ValueError):
            call(q, k, k, window, **ok)
    for window in (1.5, True, "4", None):
        with pytest.raises(TypeError):
            call(q, k, k, window, **ok)
    with pytest.raises(ValueError, match="sinks"):
        call(q, k, k, 4, -1, **ok)
    with pytest.raises(TypeError, match="scale"):
        call(q, k, k, 4, scale="x", **ok)
    with pytest.raises(TypeError, match="float32"):
        call(q.half(), k.half(), k.half(), 4, **ok)
    lens = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="query length of 1"):
        call(q, k, k, 4, lengths=lens, **ok)
    one = t(1, 4, 1, 8)
    with pytest.raises(TypeError, match="int32"):
        call(one, k, k, 4, lengths=lens.long(), **ok)
    with pytest.raises(ValueError, match="lengths"):
        call(one, k, k, 4, lengths=torch.zeros(2, dtype=torch.int32), **ok)
    with pytest.raises(ValueError, match="offset"):
        call(one, k, k, 4, lengths=lens, offset=3, **ok)
    with pytest.raises(TypeError, match="mask"):
        call(q, k, k, 4, attn_mask=t(3, 5, dtype=torch.float16), **ok)
    with pytest.raises(NotImplementedError, match="gradient"):
        call(one.clone().requires_grad_(), k, k, 4, lengths=lens, **ok)
    with pytest.raises(RuntimeError, match="CUDA"):
        call(q, k, k, 4, **ok)


def test_rotary_refusals():
    freq, _ = F.rotary_frequencies(8)
    pos = torch.arange(3)
    q, k = t(1, 4, 3, 8), t(1, 2, 3, 8)
    w = torch.ones(8)
    for call in (lambda q, k, p, f, **kw: F.rotary_embedding(q, k, p, f, **kw),
                 lambda q, k, p, f, **kw: F.qk_norm_rotary(q, k, w, w, p, f, **kw)):
        with pytest.raises(TypeError, match="Tensor"):
            call(q.numpy(), k, pos, freq)
        with pytest.raises(TypeError, match="one type"):
            call(q, k.half(), pos, freq)
        with pytest.raises(TypeError, match="float32"):
            call(q.double(), k.double(), pos, freq)
        with pytest.raises(ValueError, match="rank"):
            call(q, k[0], pos, freq)
        with pytest.raises(TypeError, match="positions"):
            call(q, k, pos.float(), freq)
        with pytest.raises(TypeError, match="inv_freq"):
            call(q, k, pos, freq.float())
        with pytest.raises(TypeError, match="interleaved"):
            call(q, k, pos, freq, interleaved=1)
        with pytest.raises(TypeError, match="amplitude"):
            call(q, k, pos, freq, amplitude="x")
        with pytest.raises(RuntimeError, match="CUDA"):
            call(q, k, pos, freq)
    with pytest.raises(TypeError, match="weights"):
        F.qk_norm_rotary(q.half(), k.half(), w.bfloat16(), w, pos, freq)
    with pytest.raises(ValueError, match="weights"):
        F.qk_norm_rotary(q, k, torch.ones(4), w, pos, freq)
    with pytest.raises(ValueError, match="key"):
        F.qk_norm_rotary(q, None, w, w, pos, freq)
    with pytest.raises(ValueError, match="eps"):
        F.qk_norm_rotary(q, k, w, w, pos, freq, eps=-1.0)
    with pytest.raises(ValueError, match="eps"):
        F.qk_norm_rotary(q, k, w, w, pos, freq, eps=math.nan)


def test_rotary_frequencies():
    f, a = F.rotary_frequencies(8, base=100.0)
    assert a == 1.0 and f.dtype == torch.float64
    assert torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64), rtol=1e-15)
    assert torch.equal(F.rotary_frequencies(8, base=100.0, scaling="linear", factor=2.0)[0], f / 2)
    n, _ = F.rotary_frequencies(8, scaling="ntk", factor=8.0)
    p, _ = F.rotary_frequencies(8)
    assert n[0] == 1.0 and math.isclose(n[-1] * 8.0, p[-1], rel_tol=1e-12)  # the slowest: interpolated by the factor
    y, amp = F.rotary_frequencies(64, scaling="yarn", factor=4.0, original_length=4096)
    p, _ = F.rotary_frequencies(64)
    turns = 4096 * p / (2 * math.pi)
    assert torch.equal(y[turns >= 32], p[turns >= 32]) and torch.equal(y[turns <= 1], p[turns <= 1] / 4)
    assert math.isclose(amp, 0.1 * math.log(4) + 1)
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, scaling="x"), dict(rotary_dim=8, base=0.0),
                dict(rotary_dim=8, scaling="yarn"), dict(rotary_dim=2, scaling="ntk")):
        with pytest.raises(ValueError):
            F.rotary_frequencies(**bad)


def test_cache_refusals():
    for bad, error in ((dict(num_pages=0), ValueError), (dict(head_dim=96), ValueError), (dict(page_size=24), ValueError),
                       (dict(page_size=8), ValueError), (dict(kv_heads=1.5), TypeError)):
        with pytest.raises(error):
            dc.KVCache4(**{**dict(num_pages=2, kv_heads=2, head_dim=64, page_size=16, device="cpu"), **bad})
    c = dc.KVCache4(2, 2, 64, page_size=16, device="cpu")
    table, n = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    k = t(1, 2, 3, 64)
    with pytest.raises(TypeError, match="int32"):
        c.append(k, k, table.long(), n)
    with pytest.raises(ValueError, match="page_table"):
        c.append(k, k, table[0], n)
    with pytest.raises(ValueError, match="start"):
        c.append(k, k, table, torch.zeros(2, dtype=torch.int32))
    with pytest.raises(TypeError, match="both"):
        c.append(k, k.half(), table, n)
    with pytest.raises(ValueError, match="key"):
        c.append(t(1, 3, 3, 64), k, table, n)
    with pytest.raises(ValueError, match="one shape"):
        c.append(k, t(1, 2, 4, 64), table, n)
    with pytest.raises(ValueError, match="query"):
        c.attention(t(1, 2, 2, 64), table, n)
    with pytest.raises(ValueError, match="multiple"):
        c.attention(t(1, 3, 1, 64), table, n)
    with pytest.raises(ValueError, match="window"):
        c.attention(t(1, 2, 1, 64), table, n, window=0)
    with pytest.raises(ValueError, match="sinks"):
        c.attention(t(1, 2, 1, 64), table, n, window=4, sinks=-1)
    with pytest.raises(NotImplementedError, match="gradient"):
        c.attention(t(1, 2, 1, 64).requires_grad_(), table, n)
    with pytest.raises(TypeError, match="float32"):
        c.attention(t(1, 2, 1, 64, dtype=torch.float64), table, n)
    with pytest.raises(ValueError, match="max_length"):
        c.read(table, n, -1)
    with pytest.raises(RuntimeError, match="CUDA"):
        c.attention(t(1, 2, 1, 64), table, n)
    with pytest.raises(RuntimeError, match="CUDA"):
        c.append(k, k, table, n)


def fake(shape, dtype=_lib.DC_F32, ptr=0x10000):
    v = _lib.DcTensor()
    v.data, v.dtype, v.ndim = ptr, dtype, len(shape)
    stride = 1
    for i in reversed(range(len(shape))):
        v.sizes[i], v.strides[i] = shape[i], stride
        stride *= max(shape[i], 1)
    return v


def test_c_entry_points_refuse_before_any_device_work():
    L = _lib.load()
    r = lambda x: None if x is None else ctypes.byref(x)
    q, k, out, lse = fake((2, 4, 8, 64)), fake((2, 2, 9, 64)), fake((2, 4, 8, 64)), fake((2, 4, 8))

    def window(window=4, sinks=0, offset=1, lens=None, q=q, mask=None, out=out, lse=lse):
        return L.dc_sdpa_window_fwd(r(q), r(k), r(k), r(mask), window, sinks, offset, r(lens), 0, 0.0, 0, r(out), r(lse),
                                    None, 0, None)

    for kw in (dict(window=0), dict(sinks=-1), dict(offset=1 << 40), dict(q=fake((2, 4, 8, 64), ptr=0x10001)), dict(out=fake((2, 4, 8, 64), ptr=0)),
               dict(lens=fake((2,), _lib.DC_I32, ptr=0), q=fake((2, 4, 1, 64)), out=fake((2, 4, 1, 64)), lse=fake((2, 4, 1))), dict(lens=fake((2,), _lib.DC_I32)),
               dict(mask=fake((3, 9), _lib.DC_BOOL)), dict(out=fake((2, 4, 8, 32))), dict(q=fake((2, 4, 8, 64), _lib.DC_BF16))):
        assert window(**kw) == _lib.DC_ERR_VALUE, kw
    pos, freq = fake((8,), _lib.DC_I64), fake((32,), _lib.DC_F64)

    def rotary(q=q, k=None, pos=pos, freq=freq, out=out, kout=None):
        return L.dc_rotary(r(q), r(k), r(pos), r(freq), 0, 1.0, 0, r(out), r(kout), None)

    assert rotary(pos=fake((9,), _lib.DC_I64)) == _lib.DC_ERR_VALUE
    assert rotary(pos=fake((3, 8), _lib.DC_I64)) == _lib.DC_ERR_VALUE
    assert rotary(freq=fake((33,), _lib.DC_F64)) == _lib.DC_ERR_VALUE
    assert rotary(freq=fake((32,))) == _lib.DC_ERR_VALUE
    assert rotary(out=fake((2, 4, 8, 64), _lib.DC_BF16)) == _lib.DC_ERR_VALUE
    assert rotary(k=fake((2, 4, 7, 64)), kout=fake((2, 4, 7, 64))) == _lib.DC_ERR_VALUE
    odd = fake((2, 4, 8, 63))
    assert rotary(q=odd, out=odd, freq=fake((4,), _lib.DC_F64)) == _lib.DC_ERR_UNSUPPORTED
    assert rotary(q=fake((2, 4, 8, 64), ptr=0)) == _lib.DC_ERR_VALUE  # no memory
    assert rotary(q=fake((2, 4, 8, 64), ptr=0x10002)) == _lib.DC_ERR_VALUE  # off its type's boundary
    negative = fake((-2, 4, -8, 64))
    assert rotary(q=negative, out=negative, pos=fake((-8,), _lib.DC_I64)) == _lib.DC_ERR_VALUE
    spread = fake((2, 4, 8, 64))
    spread.strides[1] = 0  # an output whose heads share memory
    assert rotary(out=spread) == _lib.DC_ERR_VALUE
    cache = _lib.DcCache4(0x10000, 4, 2, 64, 16)
    table, n, one = fake((2, 3), _lib.DC_I32), fake((2,), _lib.DC_I32), fake((2, 4, 1, 64))

    def attention(cache=cache, q=one, table=table, n=n, window=0, sinks=0, out=one, lse=fake((2, 4, 1))):
        return L.dc_cache4_attention(ctypes.byref(cache), r(q), r(table), r(n), window, sinks, 0, 0.0, r(out), r(lse), None, 0, None)

    for kw in (dict(cache=_lib.DcCache4(0, 4, 2, 64, 16)), dict(cache=_lib.DcCache4(0x10004, 4, 2, 64, 16)),
               dict(cache=_lib.DcCache4(0x10000, 4, 2, 64, 20)), dict(q=fake((2, 3, 1, 64))),
               dict(q=fake((2, 4, 2, 64))), dict(table=fake((2, 3), _lib.DC_I64)), dict(n=fake((3,), _lib.DC_I32)),
               dict(window=-1), dict(table=fake((2, 3), _lib.DC_I32, ptr=0)), dict(out=fake((2, 4, 1, 64), _lib.DC_BF16)), dict(lse=fake((2, 4)))):
        assert attention(**kw) == _lib.DC_ERR_VALUE, kw
    assert attention(cache=_lib.DcCache4(0x10000, 4, 2, 96, 16)) == _lib.DC_ERR_UNSUPPORTED
    assert attention(table=fake((2, 1 << 28), _lib.DC_I32)) == _lib.DC_ERR_UNSUPPORTED
    if not torch.cuda.is_available():
        assert window() == rotary() == attention() == _lib.DC_ERR_CUDA


def test_a_cache_keeps_to_its_own_memory():
    # The pages cannot be replaced under the description that the kernels get; copies get their own.
    import copy
    import io
    cache = dc.KVCache4(2, 1, 64, device="cpu")
    cache.data[1] = 7
    with pytest.raises(AttributeError):
        cache.data = torch.zeros_like(cache.data)
    twin = copy.deepcopy(cache)
    file = io.BytesIO()
    torch.save(cache, file)
    file.seek(0)
    loaded = torch.load(file, weights_only=False)
    for other in (twin, loaded):
        assert other.data.data_ptr() != cache.data.data_ptr() and torch.equal(other.data, cache.data)
        assert other._desc.data == other.data.data_ptr() and other.device == cache.device
        assert (other._desc.num_pages, other._desc.kv_heads, other._desc.head_dim, other._desc.page_size) == (2, 1, 64, 64)
    assert cache._desc.data == cache.data.data_ptr()


def window_backward(**kw):
    """dc_sdpa_window_bwd on made-up memory, with the tensors in ``kw`` in place of good ones."""
    L = _lib.load()
    big, small = (2, 4, 8, 64), (2, 2, 9, 64)
    ts = dict(go=fake(big), q=fake(big), k=fake(small), v=fake(small), out=fake(big), lse=fake((2, 4, 8)), mask=None,
              gq=fake(big), gk=fake(small), gv=fake(small))
    ts.update(kw)
    r = {name: None if x is None else ctypes.byref(x) for name, x in ts.items()}
    return L.dc_sdpa_window_bwd(r["go"], r["q"], r["k"], r["v"], r["out"], r["lse"], r["mask"], 4, 0, 1, 0, 0.0, 0, r["gq"], r["gk"],
                                r["gv"], None, 0, None)


# Made-up memory: these run only where there is no device that a call let through could touch.
without_a_device = pytest.mark.skipif(torch.cuda.is_available(), reason="passes made-up addresses")


@without_a_device
@pytest.mark.parametrize("name", ["go", "q", "k", "v", "out", "lse", "gq", "gk", "gv", "mask"])
def test_window_backward_refuses_memory_it_cannot_follow(name):
    shape = {"k": (2, 2, 9, 64), "v": (2, 2, 9, 64), "gk": (2, 2, 9, 64), "gv": (2, 2, 9, 64), "lse": (2, 4, 8),
             "mask": (8, 9)}.get(name, (2, 4, 8, 64))
    for ptr in (0, 0x10002):
        assert window_backward(**{name: fake(shape, ptr=ptr)}) == _lib.DC_ERR_VALUE
        assert "aligned" in _lib.load().dc_last_error().decode()
    if name != "mask":
        assert window_backward(**{name: None}) == _lib.DC_ERR_VALUE
    assert window_backward() == _lib.DC_ERR_CUDA


@without_a_device
def test_expanded_outputs_without_elements_are_taken():
    # torch.empty_like of an expanded tensor without elements is expanded too.
    L = _lib.load()
    r = ctypes.byref
    for shape, dim in (((3, 2, 0, 64), 0), ((0, 5, 3, 64), 1)):
        q, out = fake(shape, ptr=0), fake(shape, ptr=0)
        q.strides[dim] = out.strides[dim] = 0
        pos = fake(shape[2:3], _lib.DC_I64)
        assert L.dc_rotary(r(q), None, r(pos), r(fake((32,), _lib.DC_F64)), 0, 1.0, 0, r(out), None, None) == _lib.DC_OK


@without_a_device
def test_outputs_whose_elements_share_memory_are_refused():
    L = _lib.load()
    r = ctypes.byref

    def spread(shape, dim):
        t = fake(shape)
        t.strides[dim] = 0
        return t

    big, small, rows = (2, 4, 8, 64), (2, 2, 9, 64), (2, 4, 8)
    for dim in range(4):
        for name, shape in (("gq", big), ("gk", small), ("gv", small)):
            assert window_backward(**{name: spread(shape, dim)}) == _lib.DC_ERR_VALUE
            assert "share" in L.dc_last_error().decode()
    for name, shape in (("go", big), ("q", big), ("k", small), ("v", small), ("out", big)):
        assert window_backward(**{name: spread(shape, 1)}) == _lib.DC_ERR_CUDA  # inputs may be expanded

    def forward(out, lse):
        return L.dc_sdpa_window_fwd(r(fake(big)), r(fake(small)), r(fake(small)), None, 4, 0, 1, None, 0, 0.0, 0, r(out), r(lse),
                                    None, 0, None)

    assert forward(fake(big), fake(rows)) == _lib.DC_ERR_CUDA
    for dim in range(4):
        assert forward(spread(big, dim), fake(rows)) == _lib.DC_ERR_VALUE
    for dim in range(3):
        assert forward(fake(big), spread(rows, dim)) == _lib.DC_ERR_VALUE
    cache, one = _lib.DcCache4(0x10000, 4, 2, 64, 16), (2, 4, 1, 64)

    def attention(lse):
        return L.dc_cache4_attention(r(cache), r(fake(one)), r(fake((2, 3), _lib.DC_I32)), r(fake((2,), _lib.DC_I32)), 0, 0, 0, 0.0,
                                     r(fake(one)), r(lse), None, 0, None)

    assert attention(fake((2, 4, 1))) == _lib.DC_ERR_CUDA
    for dim in (0, 1):
        assert attention(spread((2, 4, 1), dim)) == _lib.DC_ERR_VALUE
