"""moe_linear, moe_router_select and the layer with a shared expert in calls that the documents
allow: rows so far apart that offsets pass 32 bits, the very first call of a process inside a
graph capture, and first calls from several host threads at once."""
import os
import subprocess
import sys
import threading

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.fixture(autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield
    torch.cuda.empty_cache()


def far(rows, cols, ld, dtype):
    return torch.empty((rows - 1) * ld + cols, dtype=dtype, device="cuda").as_strided((rows, cols), (ld, 1))


@pytest.mark.parametrize("kernel, T, K, N, ldx, ldw, ldy", [
    ("few", 3, 64, 20, 2 ** 30 + 2 ** 29, 2 ** 27, 2 ** 31 + 3), ("narrow", 40, 512, 40, 2 ** 26 + 8, 2 ** 26 + 8, 2 ** 26 + 5),
    ("split4n", 40, 2048, 40, 2 ** 26 + 8, 2 ** 26 + 8, 2 ** 26 + 5),
    ("pair", 2048, 64, 2400, 2 ** 21, 2 ** 20, 2 ** 21 + 8), ("pair", 2048, 64, 2400, 2 ** 10, 2 ** 20, 2 ** 21 + 1)])
def test_offsets_beyond_32_bits(moe, kernel, T, K, N, ldx, ldw, ldy):
    assert moe.linear_kernel(T, K, N) == kernel
    mats = [far(T, K, ldx, torch.float16), far(N, K, ldw, torch.float16), far(T, N, ldy, torch.float16)]
    for m in mats:
        m.copy_(torch.randint(-3, 4, m.shape, device="cuda"))
    x, w, y = mats
    want = x.double() @ w.double().t() + y.double()
    moe.moe_linear(x, w, residual=y, y=y)
    assert torch.equal(y.double(), want)


@pytest.mark.parametrize("T, ld", [(40, 2 ** 26 + 1), (1200, 2 ** 21 + 4)])
def test_select_offsets_beyond_32_bits(moe, T, ld):
    l = far(T, 64, ld, torch.float32)
    l.copy_(torch.randn((T, 64), device="cuda"))
    ids, _ = moe.moe_router_select(l, 6)
    assert torch.equal(ids.long(), l.contiguous().topk(6).indices)


FIRST = """
import torch
from _moe_loader import load
moe = load()
what = %r
T = dict(few=4, split=40, pairn=600, pair=4096, layer=300).get(what, 2000)
r = lambda *s: torch.randn(s, device="cuda").half() / s[-1] ** 0.5
x, w, wd, wr, ew = r(T, 1024), r(1024, 1024), r(1024, 512), r(16, 1024), r(16, 192, 1024)  # fp16
wide, l = r(4096, 1024), torch.randn((2000, 64), device="cuda")
ws = torch.empty(1 << 26, dtype=torch.uint8, device="cuda")
y = torch.zeros((T, 4096 if what == "pair" else 1024), dtype=torch.float16, device="cuda")
ids, wt = torch.zeros((2000, 6), dtype=torch.int32, device="cuda"), torch.zeros((2000, 6), dtype=torch.float16, device="cuda")

def call():
    if what == "select":
        moe.moe_router_select(l, 6, expert_ids=ids, weights=wt)
    elif what == "layer":
        moe.moe_shared_layer_forward(x, wr, ew, w, wd, 2, y=y, workspace=ws)
    else:
        moe.moe_linear(x, wide if what == "pair" else w, y=y)

g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    call()
g.replay()
got = [t.clone() for t in (y, ids, wt)]
for t in (y, ids, wt):
    t.zero_()
call()
assert all(torch.equal(a, b) for a, b in zip(got, (y, ids, wt)))
assert (ids if what == "select" else y).any()
assert what in ("select", "layer") or moe.linear_kernel(*x.shape, y.shape[1]).startswith(what)
"""


@pytest.mark.parametrize("what", ["few", "split", "pairn", "pair", "select", "layer"])
def test_first_call_is_captured(what):
    code = "import sys; sys.path[:0] = [%r, %r]\n" % (HERE, os.path.dirname(HERE)) + FIRST % what
    r = subprocess.run([sys.executable, "-c", code], cwd=os.path.dirname(HERE), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


def test_threads(moe):
    """Eight host threads, each on a stream of its own."""
    x, w = torch.randn((1024, 1024), device="cuda").half(), torch.randn((2048, 1024), device="cuda").half() / 32
    l = torch.randn((3000, 64), device="cuda")
    torch.cuda.synchronize()
    out = {}

    def go(k):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            r = [moe.moe_linear(x[:T], w, activation="silu", gated=True) for T in (1024, 40, 4, 300, 128)]
            r += list(moe.moe_router_select(l, 6))
            s.synchronize()
        out[k] = r

    ts = [threading.Thread(target=go, args=(k,)) for k in range(8)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    assert len(out) == 8
    assert all(torch.equal(a, b) for k in range(8) for a, b in zip(out[k], out[0]))
