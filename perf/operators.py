"""The operators around the attention path, as a user's program calls them, with their plain forms.

Four families stand beside ``scaled_dot_product_attention``: rotary positions, norms of queries and
keys with the rotation in the same pass, attention with a sliding window and visible first tokens
(training, prefill and single-token decode), and a key/value cache held in 4 bits (filling it, and the
attention of one token over it). ``run`` computes a case with elementary torch operations where ``own``
is false and with the package's operators where it is true; ``exact`` computes it in 64 bits.
"""
import math

import torch

own = False

# ------------------------------------------------------------------------------- cases ----


def listed():
    return [
        # One decode step of a batch of 64: queries of 32 heads, keys of 8, one token each.
        dict(name="rotary_token", op="rotary", batch=64, heads=32, kv_heads=8, length=1, dim=128, rotary=128,
             interleaved=False, dtype="bfloat16", scaling="none", start=8191, train=False),
        # A training step at GPT-2-small's attention shape, half of each head rotated, pairs side by side.
        dict(name="rotary_train", op="rotary", batch=8, heads=12, kv_heads=12, length=1024, dim=64, rotary=32,
             interleaved=True, dtype="float32", scaling="none", start=0, train=True),
        # Prefill of a long context with interpolated frequencies (the 32K prefill's heads).
        dict(name="rotary_long", op="rotary", batch=1, heads=16, kv_heads=16, length=32768, dim=128, rotary=128,
             interleaved=False, dtype="bfloat16", scaling="yarn", start=100000, train=False),
        # One decode step with normed queries and keys.
        dict(name="norm_token", op="norm", batch=64, heads=32, kv_heads=8, length=1, dim=128, rotary=128,
             interleaved=False, dtype="bfloat16", scaling="none", start=4000, train=False),
        # A training step with normed queries and keys, grouped heads, a length off every tile.
        dict(name="norm_train", op="norm", batch=4, heads=32, kv_heads=8, length=2047, dim=128, rotary=128,
             interleaved=False, dtype="bfloat16", scaling="none", start=0, train=True),
        # Training at GPT-2-small's attention shape with a window of a quarter of the context.
        dict(name="window_train", op="window", batch=8, heads=12, kv_heads=12, length=1024, source=1024, dim=64,
             window=256, sinks=4, mask="none", train=True),
        # Prefill of a long prompt (the 32K prefill's heads at an odd length), each row over 2048 keys.
        dict(name="window_prefill", op="window", batch=1, heads=16, kv_heads=16, length=16383, source=16383, dim=128,
             window=2048, sinks=4, mask="none", train=False),
        # One chat session's next token: latency.
        dict(name="window_token", op="window_decode", batch=1, heads=32, kv_heads=8, capacity=8192, shortest=5000,
             dim=128, window=1000, sinks=4),
        # The split-KV decode workload (64 sequences, 32 heads, 8192 cached keys), through a window.
        dict(name="window_batch", op="window_decode", batch=64, heads=32, kv_heads=32, capacity=8192, shortest=100,
             dim=128, window=2048, sinks=4),
        # Prompts of different lengths go into the cache and are read back.
        dict(name="cache_fill", op="cache_fill", batch=8, kv_heads=8, tokens=1500, shortest=700, start=0, dim=128,
             page=64, dtype="bfloat16"),
        # One session's next token over a short cache: latency.
        dict(name="cache_token", op="cache_decode", batch=1, heads=32, kv_heads=8, capacity=1024, shortest=1000,
             dim=128, page=64, dtype="bfloat16", window=0, sinks=0),
        # The split-KV decode workload over the 4-bit cache, sequences of different lengths.
        dict(name="cache_batch", op="cache_decode", batch=64, heads=32, kv_heads=32, capacity=8192, shortest=4096,
             dim=128, page=64, dtype="float32", window=0, sinks=0),
    ]


def _spread(rng, low, high):
    """A whole number from low to high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _heads(rng, most):
    kv = rng.choice([1, 2, 3, 4, 8, 12, 16])
    return min(kv * rng.choice([1, 1, 2, 4, 8]), most) // kv * kv or kv, kv


def draw(rng):
    top = {}
    for c in listed():
        w = work(c)
        b, f = top.get(_family(c), (0, 0))
        top[_family(c)] = (max(b, w["bytes"]), max(f, w["flops"]))
    while True:
        op = rng.choice(["rotary", "norm", "window", "window_decode", "cache_fill", "cache_decode"])
        heads, kv = _heads(rng, 32)
        if op in ("rotary", "norm"):
            dim = rng.choice([64, 80, 96, 128, 256])
            rot = dim if rng.random() < 0.6 else rng.choice([dim // 2, 16, 32])
            c = dict(op=op, batch=_spread(rng, 1, 64), heads=heads, kv_heads=kv, length=_spread(rng, 1, 32768), dim=dim,
                     rotary=rot, interleaved=rng.random() < 0.4, dtype=rng.choice(["float32", "bfloat16", "float16"]),
                     scaling=rng.choice(["none", "linear", "yarn"]), start=rng.choice([0, _spread(rng, 1, 1000000)]),
                     train=rng.random() < 0.6)
        elif op == "window":
            length = _spread(rng, 1, 16384)
            extra = rng.choice([0, 0, _spread(rng, 1, 4096)])
            c = dict(op=op, batch=_spread(rng, 1, 8), heads=heads, kv_heads=kv, length=length, source=length + extra,
                     dim=rng.choice([64, 64, 128, 128, 32]), window=_spread(rng, 1, 4096), sinks=rng.choice([0, 1, 4, 64, 200]),
                     mask=rng.choice(["none", "none", "padding", "bias"]), train=rng.random() < 0.6)
            if c["dim"] == 32:  # the kernels for other head dims: shorter lengths
                c["length"] = min(c["length"], 1000)
                c["source"] = min(c["source"], 2000)
        elif op == "window_decode":
            capacity = _spread(rng, 16, 32768)
            c = dict(op=op, batch=_spread(rng, 1, 64), heads=heads, kv_heads=kv, capacity=capacity,
                     shortest=rng.choice([0, 1, max(1, capacity // 2)]), dim=rng.choice([64, 128]),
                     window=_spread(rng, 1, 8192), sinks=rng.choice([0, 1, 4, 100]))
        elif op == "cache_fill":
            tokens = _spread(rng, 1, 4096)
            c = dict(op=op, batch=_spread(rng, 1, 64), kv_heads=kv, tokens=tokens,
                     shortest=rng.choice([0, tokens, max(1, tokens // 2)]), start=rng.choice([0, _spread(rng, 1, 300)]),
                     dim=rng.choice([64, 128, 256]), page=rng.choice([16, 32, 64, 128]),
                     dtype=rng.choice(["float32", "bfloat16", "float16"]))
        else:
            capacity = _spread(rng, 16, 65536)
            c = dict(op=op, batch=_spread(rng, 1, 64), heads=heads, kv_heads=kv, capacity=capacity,
                     shortest=rng.choice([0, 1, max(1, capacity // 2)]), dim=rng.choice([64, 128, 256]),
                     page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["float32", "bfloat16", "float16"]),
                     window=rng.choice([0, 0, _spread(rng, 1, 8192)]), sinks=rng.choice([0, 4, 100]))
            if not c["window"]:
                c["sinks"] = 0
        w = work(c)
        b, f = top[_family(c)]
        pairs = c["batch"] * heads * c["length"] * c["source"] if op == "window" else 0
        stored = c["batch"] * kv * c["capacity"] * c["dim"] if "capacity" in c else 0
        if w["bytes"] <= b and w["flops"] <= max(f, 1) and pairs <= 16 * 16383 ** 2 and stored <= 64 * 32 * 8192 * 128:
            return c


def _family(c):
    return {"rotary": "positions", "norm": "positions", "cache_fill": "cache_fill"}.get(c["op"], c["op"])


# -------------------------------------------------------------------------------- work ----


def _lengths(case):
    """The sequences' lengths: spread evenly from the shortest to the capacity (or token count)."""
    n, low, high = case["batch"], case["shortest"], case.get("capacity", case.get("tokens"))
    return [high] if n == 1 else [low + (high - low) * i // (n - 1) for i in range(n)]


def _visible_keys(length, window, sinks):
    """Keys that the last token of a sequence sees."""
    return length if not window or length <= window else window + min(sinks, length - window)


def _visible_pairs(case):
    off, w, s = case["source"] - case["length"], case["window"], case["sinks"]
    total = 0
    for i in range(case["length"]):
        total += _visible_keys(min(i + off + 1, case["source"]), w, s)
    return total


def work(case):
    op, size = case["op"], {"float32": 4}.get(case.get("dtype", "float32"), 2)
    if op in ("rotary", "norm"):
        rows = case["batch"] * case["length"] * (case["heads"] + case["kv_heads"])
        passes = (2 + 2) if op == "rotary" else (2 + 3)  # backward: the gradients in and out (and the inputs again)
        n = rows * case["dim"]
        per = 3 if op == "rotary" else 8
        return {"bytes": n * size * (passes if case["train"] else 2) + 8 * case["batch"] * case["length"],
                "flops": n * per * (3 if case["train"] else 1)}
    if op == "window":
        b, h, kv, l, s, d = (case[k] for k in ("batch", "heads", "kv_heads", "length", "source", "dim"))
        pairs = b * h * _visible_pairs(case)
        q, k = 4 * b * h * l * d, 4 * b * kv * s * d
        fwd = 2 * q + 2 * k
        bwd = 4 * q + 4 * k  # q, out, grad_out in, grad_q out; k, v in, grad_k, grad_v out
        return {"bytes": fwd + (bwd if case["train"] else 0), "flops": 4 * d * pairs * (3.5 if case["train"] else 1)}
    if op == "window_decode":
        keys = sum(_visible_keys(n, case["window"], case["sinks"]) for n in _lengths(case))
        d = case["dim"]
        return {"bytes": 8 * d * case["kv_heads"] * keys + 8 * d * case["batch"] * case["heads"],
                "flops": 4 * d * case["heads"] * keys}
    if op == "cache_fill":
        d, kv, b = case["dim"], case["kv_heads"], case["batch"]
        tokens = sum(_lengths(case))
        packed = d // 2 + d // 32 * 4
        # in, packed, read again, written out in 32 bits (zeros behind each sequence's end)
        out = 2 * 4 * d * kv * b * (case["start"] + case["tokens"])
        return {"bytes": 2 * kv * tokens * (d * size + 2 * packed) + out, "flops": 2 * kv * tokens * d * 6}
    keys = sum(_visible_keys(n, case["window"], case["sinks"]) for n in _lengths(case))
    d = case["dim"]
    return {"bytes": 2 * case["kv_heads"] * keys * (d // 2 + d // 32 * 4) + 2 * size * d * case["batch"] * case["heads"],
            "flops": 4 * d * case["heads"] * keys}


# ------------------------------------------------------------------------------ inputs ----


def _frequencies(rot, scaling):
    """Rotary frequencies in 64 bits and the factor of the rotated values: plain, positions
    interpolated by 4, or interpolated by 4 for the slow frequencies only."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    if scaling == "linear":
        return f / 4, 1.0
    if scaling == "yarn":
        turns = 8192 * f / (2 * math.pi)
        keep = ((turns - 1) / (32 - 1)).clamp(0, 1)
        return f * keep + f / 4 * (1 - keep), 0.1 * math.log(4) + 1.0
    return f, 1.0


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    rand = lambda *shape: torch.randn(shape, generator=g, device=dev)
    op = case["op"]
    st = dict(case=case)
    if op in ("rotary", "norm"):
        b, h, kv, l, d = (case[k] for k in ("batch", "heads", "kv_heads", "length", "dim"))
        dt = getattr(torch, case["dtype"])
        # The fused projection's output, seen as heads.
        proj = rand(b, l, (h + 2 * kv) * d).to(dt)
        q = proj[..., :h * d].view(b, l, h, d).transpose(1, 2)
        k = proj[..., h * d:(h + kv) * d].view(b, l, kv, d).transpose(1, 2)
        st["freq"], st["amplitude"] = _frequencies(case["rotary"], case["scaling"])
        st["freq"] = st["freq"].to(dev)
        # Each sequence stands at its own position.
        first = case["start"] + torch.randint(0, 100, (b, 1), generator=g, device=dev)
        st["positions"] = first + torch.arange(l, device=dev)
        if op == "norm":
            st["wq"] = (1 + 0.2 * rand(d)).to(dt)
            st["wk"] = (1 + 0.2 * rand(d)).to(dt)
        if case["train"]:
            q, k = q.detach().requires_grad_(True), k.detach().requires_grad_(True)
            st["gq"], st["gk"] = rand(b, h, l, d).to(dt), rand(b, kv, l, d).to(dt)
            if op == "norm":
                st["wq"].requires_grad_(True)
                st["wk"].requires_grad_(True)
        st["q"], st["k"] = q, k
        return st
    if op == "window":
        b, h, kv, l, s, d = (case[k] for k in ("batch", "heads", "kv_heads", "length", "source", "dim"))
        st["q"] = rand(b, l, h, d).transpose(1, 2)
        st["k"], st["v"] = rand(b, s, kv, d).transpose(1, 2), rand(b, s, kv, d).transpose(1, 2)
        st["mask"] = None
        if case["mask"] == "padding":  # sequences padded on the left: their first rows may see no key
            pad = torch.randint(0, max(1, s // 2) + 1, (b, 1, 1, 1), generator=g, device=dev)
            st["mask"] = torch.arange(s, device=dev) >= pad
        elif case["mask"] == "bias":
            st["mask"] = rand(1, h, 1, s)
        if case["train"]:
            st["go"] = rand(b, h, l, d)
            for n in ("q", "k", "v"):
                st[n].requires_grad_(True)
        return st
    lens = torch.tensor(_lengths(case), dtype=torch.int32, device=dev)
    lens = lens[torch.randperm(case["batch"], generator=g, device=dev)]
    st["lengths"] = lens
    if op == "window_decode":
        b, h, kv, s, d = (case[k] for k in ("batch", "heads", "kv_heads", "capacity", "dim"))
        st["q"] = rand(b, h, 1, d)
        st["k"] = torch.empty(b, kv, s, d, device=dev).normal_(generator=g)
        st["v"] = torch.empty(b, kv, s, d, device=dev).normal_(generator=g)
        return st
    b, kv, d, page = (case[k] for k in ("batch", "kv_heads", "dim", "page"))
    dt = getattr(torch, case["dtype"])
    if op == "cache_fill":
        t, start = case["tokens"], case["start"]
        st["key"] = (rand(b, t, kv, d) + 2 * rand(d)).to(dt).transpose(1, 2)
        st["value"] = rand(b, t, kv, d).to(dt).transpose(1, 2)
        st["starts"] = torch.full((b,), start, dtype=torch.int32, device=dev)
        st["ends"] = lens + start
        cap = start + t
    else:
        st["q"] = rand(b, case["heads"], 1, d).to(dt)
        cap = case["capacity"]
    per = -(-cap // page)
    st["table"] = torch.randperm(b * per, generator=g, device=dev).to(torch.int32).view(b, per)
    if own:
        import densecore_b200 as dc
        st["cache"] = dc.KVCache4(b * per, kv, d, page_size=page, device=dev)
    if op == "cache_decode":
        # The context: keys with an offset per channel, values around zero, one sequence at a time.
        parts = []
        for i in range(b):
            k = rand(1, kv, cap, d) + 2 * rand(d)
            v = rand(1, kv, cap, d)
            if own:
                st["cache"].append(k, v, st["table"][i:i + 1], torch.zeros(1, dtype=torch.int32, device=dev))
            else:
                parts.append(_quantise(torch.stack((k, v))))
        if not own:
            st["codes"] = torch.cat([p[0] for p in parts], 1)
            st["scale"] = torch.cat([p[1] for p in parts], 1)
            st["low"] = torch.cat([p[2] for p in parts], 1)
    return st


# ------------------------------------------------------------------------- plain forms ----


def _angles(st):
    a = st["positions"][:, None, :, None].double() * st["freq"]
    return a.cos().float() * st["amplitude"], a.sin().float() * st["amplitude"]


def _pairs(x, case):
    rot = case["rotary"]
    if case["interleaved"]:
        return x[..., 0:rot:2], x[..., 1:rot:2]
    return x[..., :rot // 2], x[..., rot // 2:rot]


def _rotate(x, cos, sin, case):
    a, b = _pairs(x, case)
    a, b = a * cos - b * sin, b * cos + a * sin
    y = x.clone()
    if case["interleaved"]:
        y[..., 0:case["rotary"]:2], y[..., 1:case["rotary"]:2] = a, b
    else:
        y[..., :case["rotary"] // 2], y[..., case["rotary"] // 2:case["rotary"]] = a, b
    return y


EPS = 1e-6


def _plain_positions(st):
    case = st["case"]
    cos, sin = _angles(st)
    dt = st["q"].dtype
    outs, grads, wgrads = [], [], []
    for x, w, go in ((st["q"], st.get("wq"), st.get("gq")), (st["k"], st.get("wk"), st.get("gk"))):
        x = x.detach().float()
        if w is not None:
            w = w.detach().float()
            r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
            n = x * r
            outs.append(_rotate(n * w, cos, sin, case).to(dt))
        else:
            outs.append(_rotate(x, cos, sin, case).to(dt))
        if go is not None:
            gy = _rotate(go.float(), cos, -sin, case)  # the transposed rotation
            if w is not None:
                wgrads.append((gy * n).sum((0, 1, 2)).to(dt))
                gn = gy * w
                gy = r * (gn - n * (gn * n).mean(-1, keepdim=True))
            grads.append(gy.to(dt))
    return outs + grads + wgrads


def _visible(rows, source, window, sinks, offset, dev):
    """rows x source: the keys that each query row sees (row i stands at key offset + i)."""
    t = rows.to(dev)[:, None] + offset
    j = torch.arange(source, device=dev)
    return (j <= t) & ((j > t - window) | (j < sinks))


def _plain_window(st):
    case = st["case"]
    q, k, v = (st[n].detach() for n in ("q", "k", "v"))
    b, h, l, d = q.shape
    kv, s = k.shape[1], k.shape[2]
    scale, offset, rep = 1 / math.sqrt(d), s - l, h // kv
    out = torch.empty(b, h, l, d, device=q.device)
    train = case["train"]
    if train:
        gq, gk, gv = torch.zeros(b, h, l, d, device=q.device), torch.zeros_like(k), torch.zeros_like(v)
    step = max(1, (1 << 28) // (rep * s))
    for r in range(0, l, step):
        rows = torch.arange(r, min(l, r + step))
        seen = _visible(rows, s, case["window"], case["sinks"], offset, q.device)
        for i in range(b):
            for m in range(kv):
                hs = slice(m * rep, (m + 1) * rep)
                qq, kk, vv = q[i, hs, r:r + step], k[i, m], v[i, m]
                x = (qq @ kk.T) * scale
                if case["mask"] == "bias":
                    x = x + st["mask"][0, hs]
                vis = seen & st["mask"][i, 0] if case["mask"] == "padding" else seen
                x = x.masked_fill(~vis, -math.inf)
                top = x.amax(-1, keepdim=True)
                p = (x - top.masked_fill(top == -math.inf, 0)).exp()
                total = p.sum(-1, keepdim=True)
                p = p / total.masked_fill(total == 0, 1)
                out[i, hs, r:r + step] = p @ vv
                if train:
                    go = st["go"][i, hs, r:r + step]
                    dp = go @ vv.T
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                    gq[i, hs, r:r + step] = ds @ kk
                    gk[i, m] += (ds.transpose(1, 2) @ qq).sum(0)
                    gv[i, m] += (p.transpose(1, 2) @ go).sum(0)
    return [out, gq, gk, gv] if train else [out]


def _attend(q, k, v, lengths, window, sinks):
    """One token per sequence: q (b, h, 1, d), k and v (b, kv, s, d), all in 32 bits."""
    b, h, _, d = q.shape
    kv, s = k.shape[1], k.shape[2]
    q = q.view(b, kv, h // kv, d)
    x = (q @ k.transpose(2, 3)) / math.sqrt(d)
    j = torch.arange(s, device=q.device)
    t = lengths[:, None] - 1
    vis = j <= t
    if window:
        vis = vis & ((j > t - window) | (j < sinks))
    x = x.masked_fill(~vis[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = (x - top.masked_fill(top == -math.inf, 0)).exp()
    total = p.sum(-1, keepdim=True)
    return ((p @ v) / total.masked_fill(total == 0, 1)).view(b, h, 1, d)


def _plain_window_decode(st):
    case = st["case"]
    n = max(1, (1 << 28) // (case["kv_heads"] * case["capacity"] * case["dim"]))
    return torch.cat([_attend(st["q"][i:i + n], st["k"][i:i + n], st["v"][i:i + n], st["lengths"][i:i + n],
                              case["window"], case["sinks"]) for i in range(0, case["batch"], n)])


GROUP = 32


def _quantise(x):
    """Groups of 32 channels in 4 bits: low = the least value rounded down to bfloat16, scale = a
    fifteenth of the range above it rounded up to bfloat16, code = the quotient rounded to nearest
    even; all in 32-bit arithmetic, and a group stands for low + scale * code."""
    x = x.float().unflatten(-1, (-1, GROUP))
    bits = x.amin(-1).view(torch.int32)
    low = torch.where((bits < 0) & ((bits & 0xFFFF) != 0), bits + 0x10000, bits) & ~0xFFFF
    low = low.view(torch.float32)
    width = (x.amax(-1) - low) / torch.full((), 15.0, device=x.device)
    scale = ((width.view(torch.int32) + 0xFFFF) & ~0xFFFF).view(torch.float32)
    codes = ((x - low[..., None]) / scale.masked_fill(scale == 0, 1)[..., None]).round()
    return codes.to(torch.uint8), scale.bfloat16(), low.bfloat16()


def _values(codes, scale, low):
    return (low.float()[..., None] + scale.float()[..., None] * codes).flatten(-2)


def _plain_cache_fill(st):
    case = st["case"]
    outs = []
    here = torch.arange(case["tokens"], device="cuda") < (st["ends"] - case["start"])[:, None]
    for x in (st["key"], st["value"]):
        y = _values(*_quantise(x)).masked_fill(~here[:, None, :, None], 0)
        full = torch.zeros(*y.shape[:2], case["start"] + case["tokens"], y.shape[3], device=y.device)
        full[:, :, case["start"]:] = y
        outs.append(full)
    return outs


def _plain_cache_decode(st):
    case = st["case"]
    n = max(1, (1 << 28) // (case["kv_heads"] * case["capacity"] * case["dim"]))
    outs = []
    for i in range(0, case["batch"], n):
        k, v = _values(st["codes"][:, i:i + n], st["scale"][:, i:i + n], st["low"][:, i:i + n])
        outs.append(_attend(st["q"][i:i + n].float(), k, v, st["lengths"][i:i + n], case["window"], case["sinks"]))
    return torch.cat(outs).to(st["q"].dtype)


# ----------------------------------------------------------------------------- one pass ----


def run(state):
    case, op = state["case"], state["case"]["op"]
    if not own:
        if op in ("rotary", "norm"):
            return _plain_positions(state)
        if op == "window":
            return _plain_window(state)
        return {"window_decode": _plain_window_decode, "cache_fill": _plain_cache_fill,
                "cache_decode": _plain_cache_decode}[op](state)
    from densecore_b200 import functional as F
    if op == "rotary":
        q, k = F.rotary_embedding(state["q"], state["k"], state["positions"], state["freq"],
                                  interleaved=case["interleaved"], amplitude=state["amplitude"])
        if case["train"]:
            grads = torch.autograd.grad((q, k), (state["q"], state["k"]), (state["gq"], state["gk"]))
            return [q.detach(), k.detach(), *grads]
        return [q, k]
    if op == "norm":
        q, k = F.qk_norm_rotary(state["q"], state["k"], state["wq"], state["wk"], state["positions"], state["freq"],
                                eps=EPS, interleaved=case["interleaved"], amplitude=state["amplitude"])
        if case["train"]:
            grads = torch.autograd.grad((q, k), (state["q"], state["k"], state["wq"], state["wk"]),
                                        (state["gq"], state["gk"]))
            return [q.detach(), k.detach(), *grads]
        return [q, k]
    if op == "window":
        out = F.sliding_window_attention(state["q"], state["k"], state["v"], case["window"], case["sinks"],
                                         attn_mask=state["mask"], enable_gqa=True)
        if case["train"]:
            grads = torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["go"])
            return [out.detach(), *grads]
        return [out]
    if op == "window_decode":
        return F.sliding_window_attention(state["q"], state["k"], state["v"], case["window"], case["sinks"],
                                          lengths=state["lengths"], enable_gqa=True)
    cache = state["cache"]
    if op == "cache_fill":
        cache.append(state["key"], state["value"], state["table"], state["starts"], state["ends"])
        return list(cache.read(state["table"], state["ends"], case["start"] + case["tokens"]))
    return cache.attention(state["q"], state["table"], state["lengths"], window=case["window"] or None,
                           sinks=case["sinks"])


# ------------------------------------------------------------------------------- exact ----


def _exact_turn(x, angle, amplitude, case):
    """The rotation as a product of complex numbers; values behind the rotated part pass through."""
    rot = case["rotary"]
    body, rest = x[..., :rot], x[..., rot:]
    shape = (-1, 2) if case["interleaved"] else (2, -1)
    z = body.unflatten(-1, shape)
    z = torch.complex(z[..., 0], z[..., 1]) if case["interleaved"] else torch.complex(z[..., 0, :], z[..., 1, :])
    z = z * torch.polar(torch.full_like(angle, amplitude), angle)
    body = torch.stack((z.real, z.imag), -1 if case["interleaved"] else -2).flatten(-2)
    return torch.cat((body, rest), -1)


def _exact_attention(q, k, v, vis, bias=None):
    x = q @ k.transpose(-1, -2) / math.sqrt(q.shape[-1])
    if bias is not None:
        x = x + bias
    x = torch.where(vis, x, torch.full_like(x, -1e300))
    w = torch.softmax(x, -1) * vis  # a row without keys: all of its weights are zero
    return w @ v


def exact(case, seed):
    op = case["op"]
    if op in ("cache_decode", "window_decode") and case["batch"] * case["kv_heads"] * case["capacity"] * case["dim"] > 3e9:
        return None
    if op == "window" and case["train"] and case["batch"] * case["heads"] * case["length"] * case["source"] > 4e9:
        return None
    global own
    kept, own = own, False
    try:
        st = prepare(case, seed)
    finally:
        own = kept
    if op in ("rotary", "norm"):
        angle = st["positions"].double()[:, None, :, None] * st["freq"]
        outs, grads, wgrads = [], [], []
        for n in "qk":
            x = st[n].detach().double().requires_grad_(True)
            leaves, y = [x], x
            if op == "norm":
                w = st["w" + n].detach().double().requires_grad_(True)
                leaves.append(w)
                y = y / (y.square().mean(-1, keepdim=True) + EPS).sqrt() * w
            y = _exact_turn(y, angle, st["amplitude"], case)
            outs.append(y.detach())
            if case["train"]:
                gs = torch.autograd.grad(y, leaves, st["g" + n].double())
                grads.append(gs[0])
                wgrads += gs[1:]
        return outs + grads + wgrads
    if op == "window":
        q, k, v = (st[n].detach().double() for n in "qkv")
        b, h, l, d = q.shape
        kv, s = k.shape[1], k.shape[2]
        out = torch.empty(b, h, l, d, dtype=torch.float64, device=q.device)
        gq, gk, gv = torch.zeros_like(out), torch.zeros_like(k), torch.zeros_like(v)
        step = max(1, (1 << 27) // s)
        for i in range(b):
            for j in range(h):
                for r in range(0, l, step):
                    rows = torch.arange(r, min(l, r + step))
                    t = (rows + s - l).to(q.device)[:, None]
                    c = torch.arange(s, device=q.device)
                    vis = (c <= t) & ((t - c < case["window"]) | (c < case["sinks"]))
                    if case["mask"] == "padding":
                        vis = vis & st["mask"][i, 0, 0]
                    bias = st["mask"][0, j].double() if case["mask"] == "bias" else None
                    leaves = [x.detach().requires_grad_(case["train"]) for x in (q[i, j, r:r + step], k[i, j * kv // h], v[i, j * kv // h])]
                    o = _exact_attention(*leaves, vis, bias)
                    out[i, j, r:r + step] = o.detach()
                    if case["train"]:
                        a, bb, cc = torch.autograd.grad(o, leaves, st["go"][i, j, r:r + step].double())
                        gq[i, j, r:r + step] = a
                        gk[i, j * kv // h] += bb
                        gv[i, j * kv // h] += cc
        return [out, gq, gk, gv] if case["train"] else [out]
    if op == "cache_fill":
        outs = []
        for x in (st["key"], st["value"]):
            full = torch.zeros(case["batch"], case["kv_heads"], case["start"] + case["tokens"], case["dim"],
                               dtype=torch.float64, device=x.device)
            y = _exact_cached(x)
            for i in range(case["batch"]):
                n = int(st["ends"][i]) - case["start"]
                full[i, :, case["start"]:case["start"] + n] = y[i, :, :n]
            outs.append(full)
        return outs
    b, h, d = case["batch"], case["heads"], case["dim"]
    kv = case["kv_heads"]
    out = torch.zeros(b, h, 1, d, dtype=torch.float64, device="cuda")
    for i in range(b):
        n = int(st["lengths"][i])
        if not n:
            continue
        c = torch.arange(n, device="cuda")
        if case["window"]:
            c = c[(c >= n - case["window"]) | (c < case["sinks"])]
        for m in range(kv):
            if op == "window_decode":
                k, v = st["k"][i, m, c].double(), st["v"][i, m, c].double()
            else:
                k, v = (st["low"][e, i, m, c].double()[..., None] +
                        st["scale"][e, i, m, c].double()[..., None] * st["codes"][e, i, m, c] for e in (0, 1))
                k, v = k.flatten(1), v.flatten(1)
            hs = slice(m * (h // kv), (m + 1) * (h // kv))
            w = torch.softmax(st["q"][i, hs, 0].double() @ k.T / math.sqrt(d), -1)
            out[i, hs, 0] = w @ v
    return out


def _exact_cached(x):
    """The cached values from the definition: bfloat16 bounds by stepping the nearest one outward,
    codes from the 32-bit quotient that the definition names."""
    x = x.float().unflatten(-1, (-1, GROUP))
    least, most = x.min(-1).values, x.max(-1).values
    one = torch.tensor(1, dtype=torch.int16, device=x.device)
    low = least.bfloat16()
    step = torch.where(low.float() > 0, -one, one)  # one bfloat16 further down
    low = torch.where(low.float() > least, (low.view(torch.int16) + step).view(torch.bfloat16), low)
    width = torch.div(most - low.float(), torch.full_like(most, 15))
    scale = width.bfloat16()
    scale = torch.where(scale.float() < width, (scale.view(torch.int16) + one).view(torch.bfloat16), scale)
    s = scale.float()[..., None]
    codes = torch.where(s > 0, (x - low.float()[..., None]) / s.clamp_min(1e-38), torch.zeros_like(x)).double().round()
    return (low.double()[..., None] + scale.double()[..., None] * codes).flatten(-2)
