"""The layer with a selecting router and a shared expert: gate, selection, expert FFN,
combine and shared expert in one run, against the same operators called one by one (the
same bits) and against the formulas in 64 bits."""
import pytest

torch = pytest.importorskip("torch")


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def make(moe, T, H, E, K, I, Is, seed):
    x, wg, ew = moe.make_inputs_torch(T, H, E, K, I, seed)
    g = torch.Generator(device="cuda").manual_seed(seed + 1)
    wr = wg.t().contiguous()
    s1 = (torch.randn((2 * Is, H), generator=g, device="cuda") / H ** 0.5).half() if Is else None
    s2 = (torch.randn((H, Is), generator=g, device="cuda") / Is ** 0.5).half() if Is else None
    bias = torch.round(torch.randn(E, generator=g, device="cuda") * 20) * 0.001
    return x, wr, ew, s1, s2, bias


SHAPES = [  # T, H, E, K, I, Is, G, topG, groupTop
    (1, 256, 16, 2, 128, 256, 1, 1, 1), (7, 264, 8, 2, 200, 136, 4, 2, 2), (130, 256, 32, 4, 64, 384, 8, 3, 2),
    (300, 512, 64, 6, 128, 256, 8, 4, 1), (513, 128, 4, 2, 72, 0, 1, 1, 1),
]


def run(moe, p, K, G, topG, groupTop, **kw):
    x, wr, ew, s1, s2, bias = p
    return moe.moe_shared_layer_forward(x, wr, ew, s1, s2, K, bias, G, topG, groupTop, "sigmoid", True, 2.5, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_layer_is_the_run_of_its_operators(moe, gpu, shape):
    T, H, E, K, I, Is, G, topG, groupTop = shape
    p = make(moe, T, H, E, K, I, Is, T)
    x, wr, ew, s1, s2, bias = p
    ids = torch.empty((T, K), dtype=torch.int32, device="cuda")
    w = torch.empty((T, K), dtype=torch.float16, device="cuda")
    ws = torch.empty(moe.moe_shared_layer_workspace_size(T, H, E, K, I, Is), dtype=torch.uint8, device="cuda")
    y = run(moe, p, K, G, topG, groupTop, expert_ids=ids, weights=w, workspace=ws)
    assert moe.device_error(ws) == 0

    logits = moe.moe_linear(x, wr, out_dtype=torch.float32)
    i1, w1 = moe.moe_router_select(logits, K, bias, G, topG, groupTop, "sigmoid", True, 2.5)
    eo = moe.moe_expert_ffn(x, i1, w1, ew)
    y1 = moe.moe_combine(eo, i1, w1)
    routed = y1.clone()
    if Is:
        hs = moe.moe_linear(x, s1, activation="silu", gated=True)
        moe.moe_linear(hs, s2, residual=y1, y=y1)
    assert torch.equal(ids, i1) and torch.equal(w, w1) and torch.equal(y, y1)
    assert torch.equal(run(moe, p, K, G, topG, groupTop), y)  # ids and weights in the workspace

    # the formulas in 64 bits, from the same ids: each fp16 tensor on the way (expert
    # hidden rows, expert outputs, weights, routed sum, shared hidden rows) adds half an
    # fp16 step of its own magnitude, taken here against the row's largest value; five of
    # them and the final rounding: 6 * 2^-11, and as much again for the sums of the hidden
    # rows' errors over I (random signs, weights of 1/sqrt(I)).
    xd, ewd = x.double(), ew.double()
    want = torch.zeros((T, H), dtype=torch.float64, device="cuda")
    score = torch.sigmoid(logits.double()).gather(1, i1.long())
    wd = 2.5 * score / score.sum(1, keepdim=True)
    for e in range(E):
        t, k = (i1 == e).nonzero(as_tuple=True)
        if t.numel():
            a = xd[t] @ ewd[e, :I].t()
            h = a * torch.sigmoid(a) * (xd[t] @ ewd[e, I:2 * I].t())
            want.index_put_((t,), wd[t, k].unsqueeze(1) * (h @ ewd[e, 2 * I:].reshape(H, I).t()), accumulate=True)
    scale = want.abs().amax(1, keepdim=True)
    assert ((routed.double() - want).abs() <= 12 * 2.0 ** -11 * scale + 2.0 ** -24).all()
    if Is:
        a = xd @ s1[:Is].double().t()
        want = want + (a * torch.sigmoid(a) * (xd @ s1[Is:].double().t())) @ s2.double().t()
        scale = scale + want.abs().amax(1, keepdim=True)
    assert ((y.double() - want).abs() <= 12 * 2.0 ** -11 * scale + 2.0 ** -24).all()


@pytest.mark.gpu
def test_layer_in_a_graph_and_empty(moe, gpu):
    T, H, E, K, I, Is = 64, 256, 16, 4, 128, 256
    p = make(moe, T, H, E, K, I, Is, 2)
    want = run(moe, p, K, 4, 2, 2)
    xb, y = torch.zeros_like(p[0]), torch.empty_like(want)
    ws = torch.empty(moe.moe_shared_layer_workspace_size(T, H, E, K, I, Is), dtype=torch.uint8, device="cuda")
    q = (xb,) + p[1:]
    run(moe, q, K, 4, 2, 2, y=y, workspace=ws)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run(moe, q, K, 4, 2, 2, y=y, workspace=ws)
    xb.copy_(p[0])
    g.replay()
    assert torch.equal(y, want)
    assert moe.device_error(ws) == 0
    assert tuple(run(moe, (p[0][:0],) + p[1:], K, 4, 2, 2).shape) == (0, H)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", SHAPES)
def test_layer_in_place(moe, gpu, shape):
    T, H, E, K, I, Is, G, topG, groupTop = shape
    p = make(moe, T, H, E, K, I, Is, T)
    want = run(moe, p, K, G, topG, groupTop)
    x = p[0].clone()
    assert run(moe, (x,) + p[1:], K, G, topG, groupTop, y=x) is x
    assert torch.equal(x, want)


@pytest.mark.gpu
def test_front_end_refuses_a_workspace_the_kernels_cannot_write(moe, gpu):
    p = make(moe, 4, 64, 8, 2, 64, 32, 1)
    n = moe.moe_shared_layer_workspace_size(4, 64, 8, 2, 64, 32)
    for ws in (torch.empty(n, dtype=torch.uint8), torch.empty(2 * n, dtype=torch.uint8, device="cuda")[::2],
               torch.empty(n, dtype=torch.float32, device="cuda"), torch.empty(n - 1, dtype=torch.uint8, device="cuda")):
        with pytest.raises(moe.MoeError):
            run(moe, p, 2, 1, 1, 1, workspace=ws)


def test_refusals_without_gpu(moe):
    L = moe.lib()
    p = 0x10000
    need = L.MoeSharedLayerWorkspaceSize(8, 64, 8, 2, 256, 128)
    assert need > L.MoeLayerWorkspaceSize(8, 64, 8, 2, 256)
    for bad in ((8, 60, 8, 2, 256, 128), (8, 64, 8, 2, 256, 12), (8, 64, 8, 2, 256, -8), (8, 64, 300, 2, 256, 128)):
        assert L.MoeSharedLayerWorkspaceSize(*bad) == 0

    def call(x=p, wr=p, rb=None, ew=p, s1=p, s2=p, y=p, ids=None, w=None, T=8, H=64, E=8, K=2, I=256, Is=128, G=1,
             topG=1, top=1, score=0, ws=p, n=need):
        return L.MoeSharedLayerForward(x, wr, rb, ew, s1, s2, y, ids, w, T, H, E, K, I, Is, G, topG, top, score, 0, 1.0,
                                       ws, n, None)

    for kw in (dict(H=60), dict(K=9), dict(Is=4), dict(G=3), dict(G=8, topG=1, K=2), dict(top=3)):
        assert call(**kw) == -2, kw
    for kw in (dict(x=None), dict(wr=None), dict(ew=None), dict(s1=None), dict(s2=None), dict(y=None), dict(ws=None)):
        assert call(**kw) == -1, kw
    assert call(n=need - 1) == -3
    assert call(score=2) == -5
    for kw in (dict(x=p + 2), dict(wr=p + 2), dict(ew=p + 8), dict(s1=p + 2), dict(s2=p + 2), dict(y=p + 2), dict(ws=p + 8),
               dict(rb=p + 2), dict(ids=p + 2), dict(w=p + 1)):
        assert call(**kw) == -6, kw


@pytest.mark.gpu
def test_front_end_refusals(moe, gpu):
    x, wr, ew, s1, s2, bias = make(moe, 4, 64, 8, 2, 64, 32, 1)
    ok = dict(x=x, w_router=wr, expert_weights=ew, shared_gate_up=s1, shared_down=s2)
    for kw in (dict(shared_down=None), dict(shared_gate_up=s1[:32].contiguous()), dict(w_router=wr.t()),
               dict(w_router=wr[:, :32].contiguous()), dict(router_bias=bias.half()), dict(scoreFunc="max"),
               dict(y=x[:2].contiguous()), dict(weights=x), dict(expert_ids=x), dict(topK=9), dict(numGroups=3)):
        with pytest.raises(moe.MoeError):
            moe.moe_shared_layer_forward(**dict(ok, **kw))
