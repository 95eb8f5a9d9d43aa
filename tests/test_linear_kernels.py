"""Which kernel moe_linear takes: the library's own answer, for the default choice and for
every value of MOE_LINEAR_TILE (read once per process, so each runs in a child process).
On the GPU, every token count again with a 16-bit y, in the kernel that was asked for."""
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

from test_linear import TOKENS, check_exact  # noqa: E402

HERE = os.path.dirname(os.path.abspath(__file__))
MODES = ["few", "narrow", "wide", "pair", "pairn", "split2", "split4", "split8", "split2n", "split4n"]
SIZES = [(8, 1), (64, 16), (72, 33), (136, 130), (264, 256), (1032, 71), (2048, 64), (520, 1000)]


def expected(mode, T, K, N, f32, gated):
    """The kernel that a forced mode gives, or None where it cannot run."""
    if mode == "few":
        return mode if T <= 8 or (T <= 16 and not gated) else None
    if mode in ("pair", "pairn", "wide"):
        return None if f32 else mode
    if mode.startswith("split"):
        S, nk = int(mode[5]), -(-K // 64)
        while S > nk:
            S //= 2
        return f"split{S}{mode[6:]}" if S > 1 else None
    return mode


def child(mode, code):
    env = dict(os.environ, MOE_LINEAR_TILE=mode, CUDA_VISIBLE_DEVICES="")
    r = subprocess.run([sys.executable, "-c", "import sys; sys.path[:0] = [%r, %r]\n%s" % (HERE, os.path.dirname(HERE), code)],
                       env=env, cwd=os.path.dirname(HERE), capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-2000:] + r.stderr[-2000:]


def test_default_choice(moe):
    f32 = torch.float32
    for args, want in (((1, 2048, 64, f32), "few"), ((16, 2048, 64), "few"), ((9, 2048, 64, None, True), "split4n"),
                       ((17, 7168, 256), "split8"), ((128, 2048, 2048), "split4n"), ((512, 2048, 2048), "pairn"),
                       ((512, 2048, 2048, f32), "narrow"), ((128, 2048, 8192, None, True), "narrow"),
                       ((128, 4096, 14336, None, True), "wide"), ((4096, 8192, 2048), "pair"),
                       ((4096, 8192, 2048, f32), "narrow")):
        assert moe.linear_kernel(*args) == want, args
    for args in ((0, 64, 8), (4, 12, 8), (4, 0, 8), (4, 64, 0), (-1, 64, 8), (1 << 31, 64, 8), (4, 64, 8, torch.int32)):
        assert moe.linear_kernel(*args) is None, args


@pytest.mark.parametrize("mode", MODES)
def test_forced_choice(mode):
    child(mode, f"""
import torch
from _moe_loader import load
from test_linear_kernels import expected, SIZES, TOKENS
moe = load()
for T in TOKENS:
    for K, N in SIZES:
        for gated in (False, True):
            for out in (None, torch.float32):
                got, want = moe.linear_kernel(T, K, N, out, gated), expected({mode!r}, T, K, N, out is not None, gated)
                assert got == want if want else got, (T, K, N, gated, out, got, want)
""")


@pytest.mark.parametrize("mode", ["pairs", "split3", "split8n", "narow", "PAIR"])
def test_unknown_mode_is_refused(mode):
    child(mode, """
from _moe_loader import load
moe = load()
p = 0x10000
assert moe.linear_kernel(64, 64, 64) is None
assert moe.lib().MoeLinear(p, p, None, None, p, 4, 64, 64, 0, 0, 0, 0, 1, 1, 0, 0, None) == -5
assert moe.lib().MoeLinear(p, p, None, None, p, 4, 12, 64, 0, 0, 0, 0, 1, 1, 0, 0, None) == -2
""")


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T", TOKENS)
def test_sixteen_bits_over_tokens(moe, T, gated):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    mode = os.environ.get("MOE_LINEAR_TILE")
    for K, N in SIZES:
        want = expected(mode, T, K, N, False, gated) if mode else None
        if want:
            assert moe.linear_kernel(T, K, N, None, gated) == want
        for dtype in (torch.float16, torch.bfloat16):
            check_exact(moe, T, K, N, dtype, dtype, gated, seed=T + K)


@pytest.mark.gpu
@pytest.mark.parametrize("mode", MODES)
def test_each_kernel_with_sixteen_bits(mode):
    env = dict(os.environ, MOE_LINEAR_TILE=mode)
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-p", "no:cacheprovider",
                        os.path.abspath(__file__), "-k", "test_sixteen_bits_over_tokens"],
                       cwd=os.path.dirname(HERE), env=env, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-2000:]
