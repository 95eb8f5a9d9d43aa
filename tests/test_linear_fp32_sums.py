"""Long sums of an fp32 y: segments of at most 512 products whatever kernel the sizes take,
so that the accuracy of a row does not hang on how many rows come with it."""
import os
import subprocess
import sys

import pytest

torch = pytest.importorskip("torch")

from test_linear import check_exact  # noqa: E402

pytestmark = pytest.mark.gpu
HERE = os.path.dirname(os.path.abspath(__file__))
SPLITS = ["split2", "split4", "split8", "split2n", "split4n"]


@pytest.fixture(autouse=True)
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


@pytest.mark.parametrize("shape", [(64, 14336, 8192), (32, 18432, 7168), (40, 32768, 4096), (64, 57344, 8192),
                                   (1024, 14336, 1024), (8, 57344, 4096), (16, 28672, 2048), (100, 14344, 500),
                                   (20, 7176, 2000)])
def test_long_sums_are_rounded(moe, shape):
    """Positive inputs: what the tensor cores cut off adds up to one side.  An instruction adds
    16 products in a few steps, each of which cuts off half an ulp on average; over a sum that
    grows from nothing, at most 2 units of 2^-24 of it are lost to 16 products (1.2 to 1.6
    seen), so 64 to a segment of 512.  The segments are added with one rounding each, and the
    partial sums of up to 16 warps or CTAs with one each."""
    T, K, N = shape
    g = torch.Generator(device="cuda").manual_seed(5)
    x = (torch.rand((T, K), generator=g, device="cuda") + 0.5).half()
    w = (torch.rand((N, K), generator=g, device="cuda") + 0.5).half()
    y = moe.moe_linear(x, w, out_dtype=torch.float32).double()
    want = x.double() @ w.double().t()
    units = (y - want).abs() / want * 2.0 ** 24
    limit = 512 / 16 * 2 + K / 512 + 16
    assert units.max().item() <= limit, (moe.linear_kernel(T, K, N, torch.float32), units.max().item(), limit)


@pytest.mark.parametrize("T", [17, 33, 64, 100, 128, 200])
def test_long_sums_exact(moe, T):
    """Whole numbers: one segment, an odd last one, two, three and many, with a k split that
    does not divide them evenly."""
    for K, N in ((512, 64), (1032, 200), (2048, 130), (3080, 64), (6152, 71), (14336, 264), (40968, 40)):
        check_exact(moe, T, K, N, torch.float16, torch.float32, seed=T + K)
        check_exact(moe, T, K, N, torch.bfloat16, torch.bfloat16, seed=T + K)
        if K < 15000:
            check_exact(moe, T, K, N, torch.bfloat16, torch.float32, True, "relu", seed=T + K)


def test_long_sums_repeat(moe):
    x = torch.randn((100, 14336), device="cuda").half()
    w = torch.randn((300, 14336), device="cuda").half()
    want = moe.moe_linear(x, w, out_dtype=torch.float32)
    for _ in range(20):
        assert torch.equal(moe.moe_linear(x, w, out_dtype=torch.float32), want)


@pytest.mark.parametrize("mode", SPLITS)
def test_each_split(mode):
    env = dict(os.environ, MOE_LINEAR_TILE=mode)
    r = subprocess.run([sys.executable, "-m", "pytest", "-q", "-x", "-m", "gpu", "-p", "no:cacheprovider",
                        os.path.abspath(__file__), "-k", "long_sums"],
                       cwd=os.path.dirname(HERE), env=env, capture_output=True, text=True, timeout=900)
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-2000:]
