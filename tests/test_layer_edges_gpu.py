"""The ends of what the operators around attention accept: no keys, bad lengths, traced calls."""
import pytest
import torch

import densecore_b200 as dc
from densecore_b200 import _lib, _native
from densecore_b200 import functional as F

pytestmark = pytest.mark.gpu


def leave_nans_behind(d):
    # The backward's scratch comes from the library's pool, which hands the next call what the last left.
    q = torch.full((1, 4, 64, d), float("nan"), device="cuda", requires_grad=True)
    F.sliding_window_attention(q, q, q, 16).sum().backward()


@pytest.mark.parametrize("precision", ["3xtf32", "tf32", "fp32"])
@pytest.mark.parametrize("d,ev", [(64, 64), (128, 128), (96, 20), (8, 72), (160, 160)])
@pytest.mark.parametrize("rows", [1, 2, 4, 127, 129])
def test_gradients_without_keys(rows, d, ev, precision):
    # No row sees a key: outputs and gradients are exactly 0, whatever lies in the scratch.
    codes = {"3xtf32": 0, "tf32": 1, "fp32": 2}
    leave_nans_behind(128 if max(d, ev) > 64 else 64)
    q, k, v = torch.randn(1, 2, rows, d, device="cuda"), torch.randn(1, 1, 0, d, device="cuda"), torch.randn(1, 1, 0, ev, device="cuda")
    out, lse = _native._sliding_window(q, k, v, 3, 1, -rows, precision=codes[precision])
    go = torch.randn_like(out)
    gq, gk, gv = _native._sliding_window_backward(go, q, k, v, out, lse, 3, 1, -rows, precision=codes[precision])
    assert (out == 0).all() and (lse == 0).all() and (gq == 0).all()
    assert gk.shape == k.shape and gv.shape == v.shape
    for mask in (torch.ones(rows, 0, dtype=torch.bool, device="cuda"), torch.zeros(1, 1, 1, 0, device="cuda")):
        leaf = q.clone().requires_grad_()
        y = F.sliding_window_attention(leaf, k, v, 3, 1, attn_mask=mask, enable_gqa=True)
        y.backward(go)
        assert (y == 0).all() and (leaf.grad == 0).all()


def test_read_reports_lengths_out_of_range():
    # Capacity 64; also where fewer positions are read than the table holds.
    status = _lib.load().dc_device_status
    cache = dc.KVCache4(4, 2, 64, page_size=32)
    table = torch.tensor([[0, 1], [2, 3], [1, 0]], dtype=torch.int32, device="cuda")
    k = torch.randn(3, 2, 64, 64, device="cuda")
    zeros = torch.zeros(3, dtype=torch.int32, device="cuda")
    cache.append(k[:2], k[:2], table[:2], zeros[:2])
    full, _ = cache.read(table, torch.full_like(zeros, 64), 64)
    status(1)
    for lengths, seen, bad in (((64, 0, 17), (64, 0, 17), 0), ((64, -7, 17), (64, 0, 17), 3), ((65, 5, 17), (64, 5, 17), 3),
                               ((2 ** 31 - 1, -2 ** 31, 0), (64, 0, 0), 3)):
        lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        for positions in (64, 40, 1, 100):
            key, value = cache.read(table, lens, positions)
            assert status(1) == bad, (lengths, positions)
            for b, n in enumerate(seen):
                n = min(n, positions)
                assert torch.equal(key[b, :, :n], full[b, :, :n]) and (key[b, :, n:] == 0).all()
                assert torch.equal(value[b], key[b])


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
@pytest.mark.parametrize("grad", [False, True])
def test_traced_calls_run_at_other_sizes(grad):
    freq, _ = F.rotary_frequencies(64, device="cuda")
    weight = torch.rand(64, device="cuda") + 0.5

    def layer(q, k, v, positions, key_positions):
        q, _ = F.qk_norm_rotary(q, None, weight, None, positions, freq)
        k, _ = F.rotary_embedding(k, None, key_positions, freq)
        return F.sliding_window_attention(q, k, v, 16, 2, enable_gqa=True)

    def inputs(b, rows, keys):
        q, k, v = (torch.randn(b, h, n, 64, device="cuda") for h, n in ((4, rows), (2, keys), (2, keys)))
        at = torch.arange(keys, device="cuda")
        return q.requires_grad_(grad), k.requires_grad_(grad), v, at[keys - rows:], at

    traced = torch.jit.trace(layer, inputs(1, 20, 33), check_trace=False)
    for sizes in ((1, 20, 33), (2, 70, 90), (1, 1, 40)):
        args = inputs(*sizes)
        got, ref = traced(*args), layer(*args)
        assert torch.equal(got, ref)
        if grad:
            go = torch.randn_like(ref)
            for x, y in zip(torch.autograd.grad(got, args[:2], go), torch.autograd.grad(ref, args[:2], go)):
                assert torch.equal(x, y)
    if not grad:
        one = torch.jit.trace(lambda q, k, n: F.sliding_window_attention(q, k, k, 16, lengths=n),
                              (torch.randn(2, 2, 1, 64, device="cuda"), torch.randn(2, 2, 50, 64, device="cuda"),
                               torch.tensor([3, 50], dtype=torch.int32, device="cuda")), check_trace=False)
        q, k = torch.randn(3, 2, 1, 64, device="cuda"), torch.randn(3, 2, 400, 64, device="cuda")
        n = torch.tensor([0, 400, 17], dtype=torch.int32, device="cuda")
        assert torch.equal(one(q, k, n), F.sliding_window_attention(q, k, k, 16, lengths=n))


WITHOUT_ROOM = """
import torch
from densecore_b200 import functional as F

q, k, v = (torch.randn(1, 16, 8192, 128, device="cuda") for _ in range(3))
small = [t[:, :2, :200].contiguous().requires_grad_() for t in (q, k, v)]


def step():
    out = F.sliding_window_attention(*small, 64)
    return [out.detach(), *torch.autograd.grad(out.sum(), small)]


want = step()
F.sliding_window_attention(q[:, :1, :700], k[:, :1, :700], v[:, :1, :700], 699)  # loads the kernels
leaves = [t.requires_grad_() for t in (q, k, v)]
out = F.sliding_window_attention(*leaves, 64)
go = torch.ones_like(out)
torch.cuda.synchronize()


def leave(mib):
    return torch.empty(torch.cuda.mem_get_info()[0] - (mib << 20), dtype=torch.uint8, device="cuda")


fill = leave(112)  # 64 for the output, 134 for the copies
with torch.no_grad():
    tight = F.sliding_window_attention(q, k, v, 2048)
assert all(torch.equal(x, y) for x, y in zip(step(), want))  # the next call is a clean one
del fill
torch.cuda.empty_cache()
fill = leave(512)  # 192 for the gradients, 537 for the copies
for _ in range(2):
    try:
        torch.autograd.grad(out, leaves, go, retain_graph=True)
        raise SystemExit("the backward found room")
    except torch.OutOfMemoryError:
        raise
    except RuntimeError as e:
        assert "memory" in str(e), e
    assert all(torch.equal(x, y) for x, y in zip(step(), want))
del fill, out, go
torch.cuda.empty_cache()
with torch.no_grad():
    roomy = F.sliding_window_attention(q, k, v, 2048)
err = (tight - roomy).norm() / roomy.norm()
assert 0 < err < 5e-6, err
assert all(torch.equal(x, y) for x, y in zip(step(), want))
print("fine")
"""


def test_a_call_without_room_leaves_the_next_alone():
    # In a process of its own: the library's pool keeps what earlier calls took.
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", WITHOUT_ROOM], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr
