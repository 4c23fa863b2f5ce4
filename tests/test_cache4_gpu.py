"""The 4-bit key/value cache. What it holds must equal the format's definition bit for bit. Its
attention is held against the formula in 64 bits on the cache's own values; the bound of a case counts:

  scores   q in two fp16 parts is off by 2^-24 of the head's largest channel, the products' sums in
           32 bits by 2^-22 of their absolute terms: d <= (2^-22 sum|q k| + 2^-24 max|q| sum|k|) scale,
           and weights by as much again, relatively, for numerator and sum
  weights  three bfloat16 parts 2^-24, two (16-bit queries) 2^-17; ex2.approx 2^-22 twice; the sums 2^-20
  output   all of it times the largest |v|; 16-bit outputs half a step more."""
import math

import pytest
import torch

import densecore_b200 as dc

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def define(x):
    """low + scale * code by the definition, one group of 32 channels at a time."""
    x = x.float().unflatten(-1, (-1, 32))
    least = x.amin(-1)
    low = least.bfloat16()
    bits = low.view(torch.int16).int()
    low = torch.where(low.float() > least, (bits + torch.where(low.float() > 0, -1, 1)).to(torch.int16).view(torch.bfloat16), low)
    width = (x.amax(-1) - low.float()) / torch.full((), 15.0, device=x.device)
    scale = width.bfloat16()
    scale = torch.where(scale.float() < width, (scale.view(torch.int16) + 1).view(torch.bfloat16), scale)
    s, lo = scale.float()[..., None], low.float()[..., None]
    codes = torch.where(s > 0, ((x - lo) / torch.where(s > 0, s, 1.0)).round(), torch.zeros_like(x))
    assert codes.nan_to_num().max() <= 15
    return (lo + s * codes).flatten(-2)


def table_for(b, tokens, page, extra=3, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    per = -(-tokens // page)
    pages = b * per + extra
    return pages, torch.randperm(pages, generator=g, device="cuda")[:b * per].to(torch.int32).view(b, per)


def i32(*x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def status():
    return dc._lib.load().dc_device_status(1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("layout", ["bhtd", "bthd", "odd"])
def test_append_and_read(dtype, dim, layout):
    b, kv, t, page = 3, 2, 75, 32
    g = torch.Generator(device="cuda").manual_seed(1)
    r = lambda *s: torch.randn(s, generator=g, device="cuda")

    def tokens():
        x = {"bhtd": lambda: r(b, kv, t, dim), "bthd": lambda: r(b, t, kv, dim).transpose(1, 2),
             "odd": lambda: r(b, kv, t, dim + 1)[..., 1:]}[layout]()
        return ((x + 3 * r(dim)) * 10 ** r(b, kv, t, 1)).to(dtype)

    pages, table = table_for(b, 200, page)
    cache = dc.KVCache4(pages, kv, dim, page_size=page)
    k, v = tokens(), tokens()
    start, end = i32(0, 13, 100), i32(75, 20, 160)
    cache.append(k, v, table, start, end)
    got = cache.read(table, end, 200)
    for x, y in zip((k, v), got):
        want = torch.zeros(b, kv, 200, dim, device="cuda")
        d = define(x)
        for i in range(b):
            n = int(end[i] - start[i])
            want[i, :, start[i]:end[i]] = d[i, :, :n]
        assert torch.equal(y, want)
    # places from `end` on, and pages of no sequence, keep what they hold
    before = cache.data.clone()
    cache.append(k * 0, v, table, start, start)
    assert torch.equal(cache.data, before)
    unused = torch.ones(pages, dtype=torch.bool, device="cuda")
    unused[table.flatten().long()] = False
    assert (cache.data[unused] == 0).all()
    # one token at a time
    one = dc.KVCache4(pages, kv, dim, page_size=page)
    for i in range(5):
        one.append(k[:, :, i:i + 1], v[:, :, i:i + 1], table, start + i)
    for x, y in zip((k, v), one.read(table, start + 5, 200)):
        for i in range(b):
            s = int(start[i])
            assert torch.equal(y[i, :, s:s + 5], define(x)[i, :, :5])
    assert status() == 0


def test_values_at_the_edges_of_the_format():
    x = torch.zeros(1, 1, 9, 64, device="cuda")
    x[0, 0, 1] = 7.3  # constants
    x[0, 0, 2] = -1e-41
    x[0, 0, 3, ::2] = 1e30
    x[0, 0, 4] = torch.linspace(1000.0, 1001.0, 64, device="cuda")
    x[0, 0, 5, 3] = math.inf
    x[0, 0, 6, 40] = math.nan
    x[0, 0, 7] = torch.linspace(-3e-39, 3e-39, 64, device="cuda")
    x[0, 0, 8, 0], x[0, 0, 8, 1] = 3e38, -3e38  # the range itself overflows
    pages, table = table_for(1, 16, 16)
    cache = dc.KVCache4(pages, 1, 64, page_size=16)
    cache.append(x, x, table, i32(0))
    y = cache.read(table, i32(9), 9)[0]
    want = define(x)
    fine = torch.tensor([0, 1, 2, 3, 4, 7], device="cuda")
    assert torch.equal(y[0, 0, fine], want[0, 0, fine])
    assert (y[0, 0, 1] - 7.3).abs().max() <= 7.3 * 2.0 ** -8
    assert y[0, 0, 5, :32].isnan().all() and (y[0, 0, 5, 32:] == 0).all()
    assert y[0, 0, 6, 32:].isnan().all() and (y[0, 0, 6, :32] == 0).all()
    assert y[0, 0, 8, :32].isnan().all()
    assert status() == 0


def fill(b, kv, cap, dim, page, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages, table = table_for(b, cap, page, seed=seed)
    cache = dc.KVCache4(pages, kv, dim, page_size=page)
    k = torch.randn(b, kv, cap, dim, generator=g, device="cuda") + 2 * torch.randn(dim, generator=g, device="cuda")
    v = torch.randn(b, kv, cap, dim, generator=g, device="cuda")
    cache.append(k, v, table, torch.zeros(b, dtype=torch.int32, device="cuda"))
    return cache, table


def check(cache, table, q, lens, window=None, sinks=0, scale=None):
    out, lse = cache.attention(q, table, lens, scale=scale, window=window, sinks=sinks, return_lse=True)
    cap = table.shape[1] * cache.page_size
    k, v = (x.double() for x in cache.read(table, lens, cap))
    b, h, _, d = q.shape
    kv = cache.kv_heads
    sc = 1 / math.sqrt(d) if scale is None else scale
    qd = q.double().view(b, kv, h // kv, d)
    s = qd @ k.transpose(2, 3) * sc
    j, t = torch.arange(cap, device="cuda"), lens[:, None].long() - 1
    vis = j <= t
    if window:
        vis = vis & ((t - j < window) | (j < sinks))
    s = torch.where(vis[:, None, None], s, -math.inf)
    some = vis.any(-1)
    p = torch.where(some[:, None, None, None], s.softmax(-1), 0.0)
    ref = (p @ v).view(b, h, 1, d)
    terms = (qd.abs() @ k.abs().transpose(2, 3)).amax().item()
    tops = (qd.abs().amax() * k.abs().sum(-1).amax()).item()
    ds = (2.0 ** -22 * terms + 2.0 ** -24 * tops) * abs(sc)
    part = 2.0 ** -24 if q.dtype == torch.float32 else 2.0 ** -17
    tol = v.abs().max().item() * (2 * ds + part + 2.0 ** -20)
    half = torch.finfo(q.dtype).eps / 2 if q.dtype != torch.float32 else 0.0
    err = (out.double() - ref).abs() - half * (ref.abs() + tol)
    assert out.dtype == q.dtype and torch.isfinite(out).all() and err.max().item() <= tol, (err.max().item(), tol)
    want = torch.where(some[:, None, None], s.logsumexp(-1), 0.0).view(b, h, 1)
    # log of a sum off by ds and 2^-20, in 32 bits
    assert (lse.double() - want).abs().max().item() <= ds + 2.0 ** -20 + 2.0 ** -22 * want.abs().max().item()
    assert (out[~some] == 0).all()
    assert status() == 0
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads", [(4, 4), (4, 2), (8, 2), (8, 1), (6, 1), (24, 2)])
def test_attention(dtype, dim, heads):
    h, kv = heads
    page, cap = 16 if dim == 64 else 48, 400
    lens = i32(0, 1, 15, 16, 17, 64, 399, 400)
    cache, table = fill(len(lens), kv, cap, dim, page)
    q = torch.randn(len(lens), h, 1, dim, device="cuda").to(dtype)
    check(cache, table, q, lens)
    check(cache, table, q, lens, window=1)
    check(cache, table, q, lens, window=50, sinks=5)
    check(cache, table, q, lens, window=20, sinks=100)
    check(cache, table, q, lens, window=10 ** 12, sinks=10 ** 12, scale=-0.1)


@pytest.mark.parametrize("b,h,kv,dim,page,cap", [(1, 8, 8, 128, 64, 9000), (3, 4, 1, 64, 128, 5003), (33, 6, 3, 128, 16, 300)])
def test_long_and_wide(b, h, kv, dim, page, cap):
    cache, table = fill(b, kv, cap, dim, page, seed=2)
    lens = torch.randint(cap // 2, cap + 1, (b,), device="cuda").to(torch.int32)
    for dtype in DTYPES:
        q = (4 * torch.randn(b, h, 1, dim, device="cuda")).to(dtype)
        check(cache, table, q, lens)
        check(cache, table, q.transpose(0, 1).contiguous().transpose(0, 1), lens, window=cap // 3, sinks=4)


def test_stale_places_and_unread_table_entries():
    # Behind the lengths the pages hold NaN and the table nonsense; neither is used.
    cache, table = fill(2, 2, 64, 128, 16)
    lens = i32(21, 40)
    nan = torch.full((2, 2, 64, 128), math.nan, device="cuda")
    cache.append(nan, nan, table, lens, i32(64, 64))
    q = torch.randn(2, 4, 1, 128, device="cuda")
    want = check(cache, table, q, lens)
    wild = table.clone()
    wild[0, 2:], wild[1, 3:] = -5, 10 ** 6
    assert torch.equal(cache.attention(q, wild, lens), want)
    assert status() == 0


def test_entries_out_of_range_are_reported_and_left_out():
    cache, table = fill(2, 1, 64, 64, 16)
    q = torch.randn(2, 1, 1, 64, device="cuda")
    lens = i32(50, 64)
    want = cache.attention(q, table, lens)
    over = cache.attention(q, table, i32(50, 65))
    assert status() == 3 and torch.equal(over, want)  # clamped to the table
    under = cache.attention(q, table, i32(50, -7))
    assert status() == 3 and (under[1] == 0).all() and torch.equal(under[0], want[0])
    bad = table.clone()
    bad[0, 1] = cache.num_pages
    got = cache.attention(q, bad, lens)
    assert status() == 3 and torch.isfinite(got).all() and torch.equal(got[1], want[1])
    k, _ = cache.read(bad, lens, 64)
    assert status() == 3 and (k[0, :, 16:32] == 0).all() and (k[0, :, :16] != 0).any()
    before = cache.data.clone()
    x = torch.randn(2, 1, 4, 64, device="cuda")
    cache.append(x, x, table, i32(-4, 64))  # before the start, behind the table
    assert status() == 3 and torch.equal(cache.data, before)
    assert status() == 0


def test_nan_and_infinite_queries_stay_in_their_rows():
    cache, table = fill(2, 2, 100, 64, 32)
    q = torch.randn(2, 4, 1, 64, device="cuda")
    lens = i32(100, 77)
    want = cache.attention(q, table, lens)
    q[0, 1, 0, 5] = math.nan
    got = cache.attention(q, table, lens)
    assert got[0, 1].isnan().all()
    keep = torch.ones(2, 4, dtype=torch.bool, device="cuda")
    keep[0, 1] = False
    assert torch.equal(got[keep], want[keep])
    big = torch.randn(2, 4, 1, 64, device="cuda") * 1e-30
    check(cache, table, big, lens)


def test_shared_pages_and_repeatability():
    cache, table = fill(1, 2, 128, 128, 32)
    both = table.repeat(2, 1)
    q = torch.randn(1, 4, 1, 128, device="cuda").repeat(2, 1, 1, 1)
    out = cache.attention(q, both, i32(128, 128))
    assert torch.equal(out[0], out[1])
    for _ in range(3):
        assert torch.equal(cache.attention(q, both, i32(128, 128)), out)
    # lengths and tables as strided views
    wide = torch.stack((both, both), 2)[..., 0]
    assert torch.equal(cache.attention(q, wide, i32(128, 9, 128, 9)[::2]), out)


def test_cache_of_more_than_four_gigabytes():
    # Page offsets pass 2^32 bytes: the last page of a 5 GB cache.
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs memory")
    page, kv, dim = 256, 8, 256
    pages = (5 << 30) // (kv * page // 16 * 20 * dim)
    cache = dc.KVCache4(pages, kv, dim, page_size=page)
    table = i32(pages - 1, 0).view(1, 2)
    x = torch.randn(1, kv, 300, dim, device="cuda")
    cache.append(x, x, table, i32(0))
    assert torch.equal(cache.read(table, i32(300), 300)[1], define(x))
    check(cache, table, torch.randn(1, 8, 1, dim, device="cuda"), i32(300))


def test_empty_calls():
    cache, table = fill(2, 2, 64, 64, 16)
    none = torch.empty(2, 0, dtype=torch.int32, device="cuda")
    q = torch.randn(2, 4, 1, 64, device="cuda")
    out, lse = cache.attention(q, none, i32(0, 0), return_lse=True)
    assert (out == 0).all() and (lse == 0).all() and status() == 0
    assert (cache.attention(q, none, i32(3, 0)) == 0).all() and status() == 3
    x = torch.randn(2, 2, 0, 64, device="cuda")
    cache.append(x, x, table, i32(0, 0))
    assert cache.read(table, i32(64, 64), 0)[0].shape == (2, 2, 0, 64)
    empty = torch.empty(0, 4, dtype=torch.int32, device="cuda")
    assert cache.attention(q[:0], empty, i32()).shape == (0, 4, 1, 64)
    assert (cache.read(table, i32(0, 5), 200)[1][0] == 0).all() and status() == 0


def test_two_threads_at_once():
    # Host threads on streams of their own, each with its cache.
    import threading
    sets = [fill(2, 2, 500, 128, 16, seed=s) for s in (1, 2)]
    q = torch.randn(2, 8, 1, 128, device="cuda")
    lens = i32(500, 77)
    want = [c.attention(q, t, lens) for c, t in sets]
    torch.cuda.synchronize()
    got, errors = [None, None], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(50):
                    got[i] = sets[i][0].attention(q, sets[i][1], lens)
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    [t.start() for t in threads], [t.join() for t in threads]
    assert not errors and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("scale", [1.0, 1.5, 1.0078125, 3e-38, 1.1e-37, 9e36, 2e37])
def test_codes_at_and_beside_ties(scale):
    # Halves of a step, and a few units in the last place beside them: to the even code, or to the near one.
    s = torch.tensor(scale).bfloat16().float().item()
    half = torch.arange(15, device="cuda") + 0.5
    x = torch.zeros(15, 9, 32, device="cuda")
    x[..., 31] = 15 * s
    tie = (half * s)[:, None]
    for step in range(9):
        y = tie.clone()
        for _ in range(abs(step - 4)):
            y = torch.nextafter(y, torch.full_like(y, math.inf if step > 4 else -math.inf))
        x[:, step, 1:31] = y
    x = torch.cat([x, -x], 0).reshape(1, 1, 270, 32).repeat(1, 1, 1, 2)  # 270 tokens of 64 channels
    pages, table = table_for(1, 270, 16)
    cache = dc.KVCache4(pages, 1, 64, page_size=16)
    cache.append(x, x, table, i32(0))
    want = define(x)
    for got in cache.read(table, i32(270), 270):
        assert torch.equal(got, want)
    assert status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("start,tokens", [(0, 1), (15, 2), (5, 31), (16, 33), (3, 127), (1, 130), (0, 517)])
def test_append_across_blocks(dtype, dim, start, tokens):
    # Runs that begin and end inside blocks of 16, pages and a kernel's run of tokens; rows 8 bytes off a
    # 16-byte boundary; neighbours on both sides keep what they hold.
    g = torch.Generator(device="cuda").manual_seed(7)
    total, kv = start + tokens + 20, 3
    pages, table = table_for(2, total, 16, seed=2)
    cache = dc.KVCache4(pages, kv, dim, page_size=16)
    old = torch.randn(2, kv, total, dim, generator=g, device="cuda").to(dtype)
    cache.append(old, -old, table, i32(0, 0))
    pad = 8 // old.element_size()
    new = torch.randn(2, tokens, kv, dim + pad, generator=g, device="cuda").to(dtype)[..., pad:].transpose(1, 2)
    cache.append(new, -new, table, i32(start, start), i32(start + tokens, start + (tokens + 1) // 2))
    for sign, got in zip((1, -1), cache.read(table, i32(total, total), total)):
        want = define(sign * old)
        d = define(sign * new)
        want[0, :, start:start + tokens] = d[0]
        want[1, :, start:start + (tokens + 1) // 2] = d[1, :, :(tokens + 1) // 2]
        assert torch.equal(got, want)
    assert status() == 0
