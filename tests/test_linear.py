"""moe_linear against the product and its epilogue in 64 bits."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def act64(z, name):
    if name == "relu":
        return z.clamp_min(0.0)
    if name == "gelu":
        return z * 0.5 * torch.special.erfc(-z * 0.5 ** 0.5)
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * (2 / np.pi) ** 0.5 * (z + 0.044715 * z ** 3))
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "sigmoid":
        return torch.sigmoid(z)
    return z


def reference(x, w, bias, act, gated, residual):
    """(y, bound on |y32 - y| before the final rounding), float64."""
    xd, wd = x.double(), w.double()
    z = xd @ wd.t()
    mag = xd.abs() @ wd.abs().t()
    if bias is not None:
        z = z + bias.double()
        mag = mag + bias.double().abs()
    # at most K + 1 roundings of 2^-24 of a partial sum no larger than the sum of magnitudes
    dz = (x.shape[1] + 1) * 2.0 ** -24 * mag
    # the activations' slopes stay below 1.13; up to 5 ulp of their own function and a
    # product or quotient, and exp's argument carries |z| half ulps
    N = w.shape[0] // 2 if gated else w.shape[0]
    a = act64(z[:, :N], act)
    own = 0.0 if act in ("none", "relu") else (12 + 4 * z[:, :N].abs()) * 2.0 ** -24
    da = 1.13 * dz[:, :N] + own * a.abs() + (0.0 if act in ("none", "relu") else 1e-37)
    if gated:
        u, du = z[:, N:], dz[:, N:]
        y = a * u
        dy = da * u.abs() + a.abs() * du + da * du + 2.0 ** -24 * y.abs()
    else:
        y, dy = a, da
    if residual is not None:
        y = y + residual.double()
        dy = dy + 2.0 ** -24 * y.abs()
    return y, dy


def make(T, K, N, dtype, otype, gated, bias, residual, seed, integers=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows = 2 * N if gated else N

    def r(*shape):
        if integers:
            return torch.randint(-3, 4, shape, generator=g, device="cuda").float()
        return torch.randn(shape, generator=g, device="cuda")

    x = r(T, K).to(dtype)
    w = (r(rows, K) / (1 if integers else K ** 0.5)).to(dtype)
    return (x, w, (r(rows)).to(dtype) if bias else None, r(T, N).to(otype) if residual else None)


def check_exact(moe, T, K, N, dtype, otype, gated=False, act="none", seed=0, bias=True, residual=True):
    """Small whole numbers: every product and sum is exact in fp32, so y is the exact value
    rounded once, bit for bit (gated products stay below 2^24 for the sizes used)."""
    x, w, b, r = make(T, K, N, dtype, otype, gated, bias, residual, seed, integers=True)
    y = moe.moe_linear(x, w, b, act, gated, r, out_dtype=otype)
    want, _ = reference(x, w, b, act, gated, r)
    assert y.dtype == otype
    bad = (y != want.to(otype)).nonzero()
    assert bad.numel() == 0, (T, K, N, dtype, otype, gated, len(bad), bad[:4].tolist())


def check_close(moe, T, K, N, dtype, otype, gated, act, bias, residual, seed=0):
    x, w, b, r = make(T, K, N, dtype, otype, gated, bias, residual, seed)
    y = moe.moe_linear(x, w, b, act, gated, r, out_dtype=otype)
    want, dy = reference(x, w, b, act, gated, r)
    tiny = 2.0 ** -25 if otype == torch.float16 else 1e-38
    tol = dy + HALF_STEP[otype] * (want.abs() + dy) + tiny
    err = (y.double() - want).abs()
    assert (err <= tol).all(), (T, K, N, dtype, otype, gated, act, (err - tol).max().item())


TOKENS = [1, 2, 3, 7, 8, 9, 15, 16, 17, 24, 31, 32, 33, 48, 63, 64, 65, 96, 127, 128, 129, 255, 257, 300]


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T", TOKENS)
def test_exact_sums_over_tokens(moe, gpu, T, gated):
    for K, N in ((8, 1), (64, 16), (72, 33), (136, 130), (264, 256), (1032, 71), (2048, 64), (520, 1000)):
        for dtype, otype in ((torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16)):
            check_exact(moe, T, K, N, dtype, otype, gated, seed=T + K)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 8192, 2048), (8, 8192, 2048), (5, 14336, 24), (16, 2048, 16384), (100, 8192, 2048),
                                   (128, 2048, 8192), (128, 7168, 256), (200, 4096, 520), (513, 2048, 1000),
                                   (777, 1416, 1411), (1024, 2048, 2048), (2000, 520, 4100), (4096, 2048, 64),
                                   (4099, 1032, 2056), (16384, 64, 8)])
def test_exact_sums_over_shapes(moe, gpu, shape):
    T, K, N = shape
    check_exact(moe, T, K, N, torch.float16, torch.float32, False, seed=1)
    check_exact(moe, T, K, N, torch.float16, torch.float16, False, "relu", seed=2, residual=False)
    check_exact(moe, T, K, N, torch.bfloat16, torch.bfloat16, False, seed=3, bias=False)
    check_exact(moe, T, K, N, torch.float16, torch.float16, True, "relu", seed=4, bias=False, residual=False)


@pytest.mark.gpu
@pytest.mark.parametrize("per_sm, more", [(16, -1), (16, 1), (32, 0), (32, 1), (32, 17), (48, 5), (64, 0), (64, 1), (64, 33)])
def test_exact_sums_where_rows_per_warp_change(moe, gpu, per_sm, more):
    # a few tokens take one or two blocks of w rows per warp, by how many waves N makes
    N = per_sm * torch.cuda.get_device_properties(0).multi_processor_count + more
    for T in (1, 5, 8):
        check_exact(moe, T, 1032, N, torch.float16, torch.float32, seed=T)
        check_exact(moe, T, 264, N, torch.bfloat16, torch.bfloat16, act="relu", seed=T + 8)


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid"])
@pytest.mark.parametrize("gated", [False, True])
def test_activations(moe, gpu, act, gated):
    for T, K, N in ((1, 64, 40), (6, 256, 96), (40, 136, 130), (150, 72, 257), (400, 256, 300)):
        for dtype in (torch.float16, torch.bfloat16):
            for otype in (dtype, torch.float32):
                check_close(moe, T, K, N, dtype, otype, gated, act, True, True, seed=T)
                check_close(moe, T, K, N, dtype, otype, gated, act, False, False, seed=T + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 14336, 64), (8, 8192, 300), (16, 14336, 40), (100, 14336, 64), (300, 8192, 256),
                                   (700, 14336, 1000), (4096, 4096, 64)])
def test_fp32_sums_are_rounded(moe, gpu, shape):
    """An fp32 y over many products: the tensor cores cut their sums off, so a sum of n
    products of one sign is off by up to n / 16 half ulps to one side.  Segments of at most
    512 products bound that by 32 + (their number) roundings of 2^-24: positive inputs show
    it, where a single accumulator over K = 14336 is off by hundreds."""
    T, K, N = shape
    g = torch.Generator(device="cuda").manual_seed(5)
    x = (torch.rand((T, K), generator=g, device="cuda") + 0.5).half()
    w = (torch.rand((N, K), generator=g, device="cuda") + 0.5).half()
    y = moe.moe_linear(x, w, out_dtype=torch.float32).double()
    want = x.double() @ w.double().t()
    # a k split leaves at most K / 2 to one CTA, which has 4 accumulators: segments of up to
    # K / 8 products, each 16 of them cut off by at most 2 units of 2^-24 of the sum
    seg = max(512, K // 8)
    rel = (seg / 16 * 2 + K / 512 + 8) * 2.0 ** -24
    assert ((y - want).abs() <= rel * want).all(), ((y - want) / want).abs().max().item() * 2 ** 24


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 9, 50, 200])
def test_activation_range(moe, gpu, T):
    """Sums from far below to far above zero: identity weights, x over a wide range."""
    K = 64
    x = torch.linspace(-60, 60, T * K, device="cuda").view(T, K).half()
    w = torch.eye(K, device="cuda").half()
    for act in ("relu", "gelu", "gelu_tanh", "silu", "sigmoid"):
        y = moe.moe_linear(x, w, activation=act, out_dtype=torch.float32).double()
        z = x.double()
        want = act64(z, act)
        # relative, down to where fp32 leaves its normal range; gelu's tail: Phi(z) ~
        # e^(-z^2/2) carries z^2 half ulps of its argument
        rel = (16 + 4 * z.abs() + 2 * z * z) * 2.0 ** -24
        if act == "gelu_tanh":  # exp's argument u takes up to 7 roundings
            rel = rel + 7 * 2.0 ** -24 * (1.6 * (z + 0.044715 * z ** 3)).abs()
        assert ((y - want).abs() <= rel * want.abs() + 2e-37).all(), act


@pytest.mark.gpu
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("T", [1, 12, 40, 130, 700])
def test_strides_and_neighbours(moe, gpu, T, gated):
    """Padded rows everywhere, NaN in what must not be read, and what must not be written
    stays as it was; y as its own residual."""
    nan = float("nan")
    for K, N in ((72, 40), (200, 131)):
        for dtype, otype, pad in ((torch.float16, torch.float16, 8), (torch.bfloat16, torch.float32, 24),
                                  (torch.float16, torch.float16, 3)):
            x, w, b, r = make(T, K, N, dtype, otype, gated, True, True, T + K, integers=True)
            want, _ = reference(x, w, b, "none", gated, r)
            xs = torch.full((T + 2, K + 16), nan, dtype=dtype, device="cuda")
            xs[1:-1, 8:-8] = x
            ws = torch.full((w.shape[0] + 1, K + 8), nan, dtype=dtype, device="cuda")
            ws[:-1, :-8] = w
            rs = torch.full((T + 1, N + pad), nan, dtype=otype, device="cuda")
            rs[:-1, pad:] = r
            ys = torch.full((T + 2, N + 2 * pad), 77.0, dtype=otype, device="cuda")
            out = moe.moe_linear(xs[1:-1, 8:-8], ws[:-1, :-8], b, "none", gated, rs[:-1, pad:], y=ys[1:-1, pad:-pad])
            assert out.data_ptr() == ys[1:-1, pad:-pad].data_ptr()
            assert torch.equal(ys[1:-1, pad:-pad], want.to(otype))
            ys[1:-1, pad:-pad] = 77.0
            assert (ys == 77.0).all()
            ys[1:-1, pad:-pad] = r
            own = ys[1:-1, pad:-pad]
            moe.moe_linear(xs[1:-1, 8:-8], ws[:-1, :-8], b, "none", gated, own, y=own)
            assert torch.equal(own, want.to(otype))


@pytest.mark.gpu
def test_infinities_and_nan_stay_in_their_rows(moe, gpu):
    for T in (3, 40, 300):
        x, w, _, _ = make(T, 136, 70, torch.float16, torch.float16, False, False, False, 1, integers=True)
        x[1, 5] = float("nan")
        w[7] = 1.0
        x[2] = 1.0
        x[2, 9] = float("inf")
        y = moe.moe_linear(x, w, out_dtype=torch.float32)
        assert torch.isnan(y[1]).all()
        assert y[2, 7] == float("inf")
        rest = [0] + list(range(3, T))
        assert torch.equal(y[rest].double(), x[rest].double() @ w.double().t())


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 10, 100, 600])
def test_repeatable_streams_and_graphs(moe, gpu, T):
    x, w, b, r = make(T, 1024, 640, torch.float16, torch.float16, True, True, True, 3)
    want = moe.moe_linear(x, w, b, "silu", True, r)
    for _ in range(3):
        assert torch.equal(moe.moe_linear(x, w, b, "silu", True, r), want)
    # two streams at once, each several calls
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs += [moe.moe_linear(x, w, b, "silu", True, r) for _ in range(4)]
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(o, want) for o in outs)
    # two captured graphs, replayed on different streams at the same time
    graphs = []
    for i in range(2):
        xb, y = torch.zeros_like(x), torch.empty_like(want)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            moe.moe_linear(xb, w, b, "silu", True, r, y=y)
            moe.moe_linear(xb, w, b, "silu", True, y, y=y)
        graphs.append((g, xb, y))
    for scale in (1.0, -0.5):
        torch.cuda.synchronize()
        for (g, xb, y), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                xb.copy_(x * scale)
                g.replay()
        torch.cuda.synchronize()
        one = moe.moe_linear(x * scale, w, b, "silu", True, r)
        two = moe.moe_linear(x * scale, w, b, "silu", True, one)
        assert torch.equal(graphs[0][2], two) and torch.equal(graphs[1][2], two)


@pytest.mark.gpu
def test_empty_batch(moe, gpu):
    w = torch.zeros((24, 16), dtype=torch.float16, device="cuda")
    y = moe.moe_linear(torch.zeros((0, 16), dtype=torch.float16, device="cuda"), w)
    assert tuple(y.shape) == (0, 24)


def test_refusals_without_gpu(moe):
    L = moe.lib()
    p = 0x10000

    def call(x=p, w=p, b=None, r=None, y=p, T=4, K=16, N=8, ldx=0, ldw=0, ldr=0, ldy=0, dt=1, ot=1, act=0, gated=0):
        return L.MoeLinear(x, w, b, r, y, T, K, N, ldx, ldw, ldr, ldy, dt, ot, act, gated, None)

    for kw in (dict(T=-1), dict(K=0), dict(K=12), dict(N=0), dict(ldx=8), dict(ldw=8), dict(ldy=7), dict(r=p + 64, ldr=4),
               dict(ldx=-8), dict(T=1 << 31), dict(N=1 << 31), dict(K=1 << 31), dict(r=p, ldr=16), dict(ldx=1 << 40)):
        assert call(**kw) == -2, kw
    for kw in (dict(dt=0), dict(dt=3), dict(ot=27), dict(dt=27, ot=1), dict(ot=3), dict(act=6), dict(act=-1)):
        assert call(**kw) == -5, kw
    for kw in (dict(x=None), dict(w=None), dict(y=None)):
        assert call(**kw) == -1, kw
    for kw in (dict(x=p + 8), dict(w=p + 2), dict(ldx=20), dict(ldw=28), dict(b=p + 1), dict(y=p + 1),
               dict(y=p + 2, ot=0), dict(r=p + 1)):
        assert call(**kw) == -6, kw
    assert call(T=0) == 0
    assert call(T=0, x=None, w=None, y=None) == 0


def test_front_end_refusals_without_gpu(moe):
    x = torch.zeros((2, 8), dtype=torch.float16)
    with pytest.raises(moe.MoeError):
        moe.moe_linear(x, x)


@pytest.mark.gpu
def test_front_end_refusals(moe, gpu):
    h = dict(dtype=torch.float16, device="cuda")
    x, w = torch.zeros((4, 16), **h), torch.zeros((24, 16), **h)
    bad = [dict(x=x.float()), dict(x=x[0]), dict(w=w.bfloat16()), dict(w=w[:, :8]), dict(w=w.cpu()), dict(w=w[:23], gated=True),
           dict(x=torch.zeros((16, 4), **h).t()), dict(x=x[:1].expand(4, 16)), dict(bias=torch.zeros(23, **h)),
           dict(bias=torch.zeros(24, device="cuda")), dict(residual=torch.zeros((4, 23), **h)),
           dict(residual=torch.zeros((1, 24), **h).expand(4, 24)), dict(residual=torch.zeros((4, 24), device="cuda"),
                                                                        y=torch.zeros((4, 24), **h)),
           dict(y=torch.zeros((1, 24), **h).expand(4, 24)), dict(y=torch.zeros((4, 24), **h).bfloat16()),
           dict(activation="tanh"), dict(out_dtype=torch.bfloat16), dict(out_dtype=torch.float64),
           dict(x=torch.zeros((4, 17), **h)[:, 1:]), dict(x=torch.zeros((4, 12), **h), w=torch.zeros((24, 12), **h))]
    for kw in bad:
        kw = dict(dict(x=x, w=w), **kw)
        kw["weight"] = kw.pop("w")
        with pytest.raises(moe.MoeError):
            moe.moe_linear(**kw)
