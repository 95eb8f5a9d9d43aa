"""moe_router_select against the operator's definition in 64 bits: ids exactly, weights
within the roundings of their type."""
import ctypes

import numpy as np
import pytest

torch = pytest.importorskip("torch")

INF = float("inf")


def reference(logits, K, bias=None, G=1, topG=1, groupTop=1, score="softmax", renorm=False, scale=1.0):
    """Token by token from the definition, float64.  Returns ids [T,K], weights [T,K]."""
    x = logits.detach().cpu().double().numpy()
    b = None if bias is None else bias.detach().cpu().double().numpy()
    T, E = x.shape
    ids = np.zeros((T, K), np.int32)
    wts = np.zeros((T, K))
    for t in range(T):
        l = x[t]
        opened = l > -INF  # False for NaN too
        s = np.zeros(E)
        if score == "softmax":
            if opened.any():
                m = l[opened].max()
                e = np.zeros(E)
                e[opened] = [1.0 if v == m else np.exp(v - m) for v in l[opened]]
                s = e / e.sum()
        else:
            with np.errstate(over="ignore"):
                s[opened] = 1.0 / (1.0 + np.exp(-l[opened]))
        if b is not None:
            opened = opened & (b > -INF)
            key = np.where(opened, s + np.where(b > -INF, b, 0.0), -INF)
        elif groupTop == 1 or G == 1:
            key = np.where(opened, l, -INF)  # scores order as their logits do
        else:
            key = np.where(opened, s, -INF)
        if G > 1:
            size = E // G
            value = np.empty(G)
            for g in range(G):
                k = sorted(key[g * size:(g + 1) * size], reverse=True)
                value[g] = k[0] + (k[1] if groupTop == 2 and k[1] > -INF else 0.0)
            stay = sorted(range(G), key=lambda g: (-value[g], g))[:topG]
            for g in range(G):
                if g not in stay:
                    key[g * size:(g + 1) * size] = -INF
        order = sorted(range(E), key=lambda e: (-key[e], e))[:K]
        ids[t] = order
        w = np.array([s[e] if key[e] > -INF else 0.0 for e in order])
        if renorm and (key[order] > -INF).any():
            live = [e for e in order if key[e] > -INF]
            if score == "softmax":
                m = max(l[e] for e in live)
                r = {e: 1.0 if l[e] == m else np.exp(l[e] - m) for e in live}
            else:  # scores over their largest, so that none is lost to underflow
                with np.errstate(over="ignore"):
                    ls = {e: -np.log1p(np.exp(-l[e])) if l[e] > -700 else l[e] for e in live}
                m = max(ls.values())
                r = {e: np.exp(ls[e] - m) for e in live}
            tot = sum(r.values())
            w = np.array([r[e] / tot if e in r else 0.0 for e in order])
        wts[t] = w * scale
    return ids, wts


def check(moe, logits, K, wtype=None, **kw):
    kr = dict(kw)
    w0 = None
    if wtype is torch.float32:
        w0 = torch.full((logits.shape[0], K), 7.0, dtype=torch.float32, device="cuda")
    names = dict(G="numGroups", topG="topGroups", groupTop="groupTop", score="scoreFunc", renorm="renormalize",
                 scale="scale", bias="bias")
    call = {names[k]: v for k, v in kr.items()}
    rid, rw = reference(logits, K, **kw)
    judge(*moe.moe_router_select(logits, K, weights=w0, **call), rid, rw)
    # the same rows many times over: large batches share a warp between tokens
    T = logits.shape[0]
    n = -(-1100 // T)
    many = logits.repeat(n, 1)
    w0 = None if w0 is None else w0.repeat(n, 1)
    judge(*moe.moe_router_select(many, K, weights=w0, **call), np.tile(rid, (n, 1)), np.tile(rw, (n, 1)))


def judge(ids, w, rid, rw):
    torch.cuda.synchronize()
    assert ids.dtype == torch.int32 and tuple(ids.shape) == rid.shape
    got = ids.cpu().numpy()
    bad = np.nonzero((got != rid).any(axis=1))[0]
    assert bad.size == 0, (len(bad), bad[:5], got[bad[:3]], rid[bad[:3]])
    # Roundings of a weight (relative): l - m half an ulp of at most D = 64 each in the
    # numerator and in the sum, exp 2 ulp each, at most 16 sum steps, a division, a scale.
    # 2 * 64 + 2 * 4 + 16 + 2 = 154 halves of 2^-23; fp16 adds half its step, and below
    # 2^-14 its absolute half step 2^-25.
    rel = 154 * 2.0 ** -24
    tol = rel * np.abs(rw) + 1e-38
    if w.dtype == torch.float16:
        tol = tol + 2.0 ** -11 * np.abs(rw) * (1 + rel) + 2.0 ** -25
    err = np.abs(w.double().cpu().numpy() - rw)
    assert (err <= tol).all(), (err - tol).max()


@pytest.fixture
def gpu():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def draw(T, E, dtype, seed, spread=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((T, E), generator=g) * spread).to(dtype).cuda()


def steps_bias(E, seed):
    """As a balancing rule leaves it: multiples of a small step, so experts share values."""
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(-40, 41, (E,), generator=g).float() * 0.001).cuda()


SHAPES = [  # T, E, K, G, topG, groupTop
    (1, 1, 1, 1, 1, 1), (1, 256, 8, 8, 4, 2), (3, 5, 2, 1, 1, 1), (130, 64, 6, 1, 1, 1), (65, 60, 4, 4, 2, 1),
    (200, 256, 8, 8, 4, 2), (77, 256, 8, 1, 1, 1), (50, 160, 6, 8, 3, 1), (33, 128, 8, 4, 2, 2), (9, 8, 8, 1, 1, 1),
    (40, 16, 2, 4, 1, 2), (21, 255, 7, 17, 5, 2), (21, 255, 8, 3, 1, 1), (31, 256, 8, 32, 1, 1), (30, 252, 8, 9, 4, 2),
    (64, 7, 3, 7, 4, 1), (20, 31, 8, 31, 8, 1), (500, 32, 4, 2, 1, 2), (17, 250, 5, 5, 2, 2), (64, 24, 8, 8, 4, 2),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_against_definition(moe, gpu, shape, dtype):
    T, E, K, G, topG, groupTop = shape
    for i, (score, bias, renorm, scale, wtype) in enumerate([
            ("softmax", False, False, 1.0, None), ("softmax", True, True, 1.5, torch.float32),
            ("sigmoid", False, True, 2.5, torch.float32), ("sigmoid", True, True, 2.5, None),
            ("sigmoid", True, False, 1.0, torch.float32)]):
        check(moe, draw(T, E, dtype, 100 * i + E), K, wtype, bias=steps_bias(E, i) if bias else None, G=G, topG=topG,
              groupTop=groupTop, score=score, renorm=renorm, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_closer_than_32_bits_tell_apart(moe, gpu, score):
    """Neighbouring fp32 logits, shuffled: their scores differ by less than an fp32 ulp,
    with and without a constant bias, alone and inside groups."""
    g = torch.Generator().manual_seed(5)
    T, E, K = 64, 64, 8
    base = torch.tensor([2.5, -1.0, 6.0, 0.1] * (T // 4)).view(T, 1)
    ulp = torch.tensor(np.spacing(np.float32(base.numpy())))
    order = torch.stack([torch.randperm(E, generator=g) for _ in range(T)])
    logits = (base.double() + order.double() * ulp.double()).float().cuda()
    for bias in (None, torch.full((E,), 0.25).cuda()):
        for renorm in (False, True):
            check(moe, logits, K, torch.float32, bias=bias, score=score, renorm=renorm)
            check(moe, logits, K, torch.float32, bias=bias, score=score, renorm=renorm, G=8, topG=3, groupTop=2)
            check(moe, logits, K, torch.float32, bias=bias, score=score, renorm=renorm, G=8, topG=3, groupTop=1)
    # one group of 15, one lane's work, that holds every slot and what comes after
    order = torch.stack([torch.randperm(255, generator=g) for _ in range(T)])
    logits = (base.double() + order.double() * ulp.double()).float().cuda()
    for K in (6, 7, 8):
        for bias in (None, torch.full((255,), 0.25).cuda()):
            check(moe, logits, K, torch.float32, bias=bias, score=score, G=17, topG=1, groupTop=2)
            check(moe, logits, K, torch.float32, bias=bias, score=score, G=17, topG=1, groupTop=1)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties_go_to_the_lower_id(moe, gpu, score):
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        g = torch.Generator().manual_seed(6)
        logits = torch.randint(0, 3, (100, 48), generator=g).to(dtype).cuda()
        for bias in (None, torch.zeros(48).cuda(), steps_bias(48, 3)):
            check(moe, logits, 6, bias=bias, score=score)
            check(moe, logits, 6, bias=bias, score=score, G=6, topG=2, groupTop=2)
        check(moe, torch.zeros((5, 256), dtype=dtype, device="cuda"), 8, G=8, topG=4, groupTop=2, score=score)
        # the score of +0 and -0 is the same
        check(moe, torch.tensor([[-0.0, 0.0, -0.0, 0.0]], dtype=dtype).cuda(), 4, score=score)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_masked_experts_and_rows(moe, gpu, score, dtype):
    """-inf and NaN logits, -inf and NaN biases, rows with nothing left, rows with fewer
    open experts than slots, the types' lowest values, +inf."""
    T, E, K = 40, 32, 6
    lowest = torch.finfo(dtype).min
    l = draw(T, E, dtype, 9)
    l[0] = -INF
    l[1] = float("nan")
    l[2, 3:] = -INF
    l[3, 5:] = float("nan")
    l[4] = lowest
    l[5, ::2] = lowest
    l[6, 4] = INF
    l[7, [4, 9, 31]] = INF
    l[8, :8] = -INF
    l[9, [0, 31]] = torch.finfo(dtype).max
    l[10:20, 7] = -INF
    bias = steps_bias(E, 1)
    bias[3] = -INF
    bias[11] = float("nan")
    bias[12] = -1e30
    for b in (None, bias):
        for renorm in (False, True):
            check(moe, l, K, bias=b, score=score, renorm=renorm)
            check(moe, l, K, torch.float32, bias=b, score=score, renorm=renorm, G=4, topG=2, groupTop=2)
            check(moe, l, K, bias=b, score=score, renorm=renorm, G=4, topG=1, groupTop=1)
    shut = torch.full((E,), -INF).cuda()
    check(moe, l, K, bias=shut, score=score, renorm=True)
    check(moe, l, K, bias=shut, score=score, renorm=True, G=4, topG=2, groupTop=2)


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_groups_with_few_open_experts(moe, gpu, score):
    """Random masks that leave groups with none, one or a few open experts, by the logit, the
    bias or both; scores near 1, near a half and near 0."""
    for i, (T, E, K, G, topG, groupTop) in enumerate([(120, 64, 8, 8, 2, 2), (100, 160, 8, 32, 13, 2), (100, 256, 5, 16, 6, 2),
                                                      (100, 250, 8, 5, 3, 2), (100, 60, 4, 4, 2, 1), (100, 64, 7, 4, 3, 2)]):
        for off in (8.0, 0.0, -6.0):
            g = torch.Generator().manual_seed(10 * i)
            l = torch.randn((T, E), generator=g) * 1.5 + off
            keep = torch.rand((T, E), generator=g) < torch.rand((T, 1), generator=g)
            l = torch.where(keep, l, -INF).cuda()
            b = steps_bias(E, i)
            for dtype in (torch.float32, torch.bfloat16):
                check(moe, l.to(dtype), K, torch.float32, G=G, topG=topG, groupTop=groupTop, score=score, renorm=True)
            b[torch.randperm(E, generator=g)[: E // 2].cuda()] = -INF
            check(moe, l, K, torch.float32, bias=b, G=G, topG=topG, groupTop=groupTop, score=score)


@pytest.mark.gpu
def test_small_scores_keep_their_ratio(moe, gpu):
    """Sigmoids that underflow in 32 bits still renormalise to their ratio."""
    g = torch.Generator().manual_seed(3)
    l = (torch.rand((50, 40), generator=g) * 8 - torch.linspace(0, 190, 50).view(50, 1)).cuda()
    check(moe, l, 5, torch.float32, score="sigmoid", renorm=True)
    check(moe, l, 5, torch.float32, score="sigmoid", renorm=True, bias=torch.zeros(40).cuda())
    check(moe, l, 5, torch.float32, score="softmax", renorm=True, bias=torch.zeros(40).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_scores_from_one_to_underflow(moe, gpu, score):
    """Logits over a hundred units, so that scores of one row lie between 1 and what fp32
    cannot hold, beside biases of a thousandth: every comparison among the best must agree
    with every other, or a slot stays unwritten."""
    for i, (T, E, K, G, topG, groupTop) in enumerate([(150, 64, 8, 1, 1, 1), (120, 64, 8, 16, 6, 1), (100, 256, 8, 8, 4, 2),
                                                      (100, 250, 7, 5, 3, 2), (100, 128, 4, 2, 2, 2),
                                                      (150, 255, 8, 17, 1, 2), (150, 255, 7, 17, 1, 2)]):
        g = torch.Generator().manual_seed(i)
        l = (torch.randn((T, E), generator=g) * 20 - 30 + 10 * (i % 3)).cuda()
        b = (torch.randn(E, generator=g) * 10.0 ** -(3 + i % 3)).cuda()
        for renorm in (False, True):
            check(moe, l, K, torch.float32, bias=b, G=G, topG=topG, groupTop=groupTop, score=score, renorm=renorm)


@pytest.mark.gpu
def test_strided_unaligned_and_repeatable(moe, gpu):
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        wide = torch.full((90, 75), float("nan"), dtype=dtype, device="cuda")
        for off, E in ((0, 64), (1, 64), (3, 60), (8, 64), (4, 56)):
            wide[:, off:off + E] = draw(90, E, dtype, off + E)
            check(moe, wide[:, off:off + E], 5, score="sigmoid", renorm=True, bias=steps_bias(E, off))
            check(moe, wide[::2, off:off + E], 5)
            wide.fill_(float("nan"))
    l = draw(3000, 256, torch.float32, 1)
    b = steps_bias(256, 2)
    first = moe.moe_router_select(l, 8, b, 8, 4, 2, "sigmoid", True, 2.5)
    for _ in range(3):
        again = moe.moe_router_select(l, 8, b, 8, 4, 2, "sigmoid", True, 2.5)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    # one row at a time gives what the batch gives
    for t in (0, 1234, 2999):
        i1, w1 = moe.moe_router_select(l[t:t + 1], 8, b, 8, 4, 2, "sigmoid", True, 2.5)
        assert torch.equal(i1[0], first[0][t]) and torch.equal(w1[0], first[1][t])


@pytest.mark.gpu
def test_many_rows(moe, gpu):
    """Larger batches, against the same definition in torch's 64 bits (no ties here)."""
    T, E, K = 20011, 256, 8
    l = draw(T, E, torch.float32, 21)
    b = (torch.randn(E, generator=torch.Generator().manual_seed(2)) * 0.05).cuda()
    ids, w = moe.moe_router_select(l, K, b, scoreFunc="sigmoid", renormalize=True, scale=2.5)
    s = torch.sigmoid(l.double())
    rid = (s + b.double()).topk(K, dim=1).indices
    assert torch.equal(ids.long(), rid)
    rw = s.gather(1, rid)
    rw = 2.5 * rw / rw.sum(1, keepdim=True)
    assert ((w.double() - rw).abs() <= rw * (2.0 ** -11 + 1e-5)).all()
    ids, w = moe.moe_router_select(l, K)
    assert torch.equal(ids.long(), l.topk(K, dim=1).indices)


@pytest.mark.gpu
def test_streams_graphs_and_empty(moe, gpu):
    l = draw(300, 64, torch.float32, 4)
    want = moe.moe_router_select(l, 6, renormalize=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = moe.moe_router_select(l, 6, renormalize=True)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    buf = torch.zeros_like(l)
    ids = torch.full((300, 6), -1, dtype=torch.int32, device="cuda")
    w = torch.zeros((300, 6), dtype=torch.float16, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        moe.moe_router_select(buf, 6, renormalize=True, expert_ids=ids, weights=w)
    for seed in (4, 5):
        buf.copy_(draw(300, 64, torch.float32, seed))
        g.replay()
        a, c = moe.moe_router_select(buf, 6, renormalize=True)
        assert torch.equal(ids, a) and torch.equal(w, c)
    i0, w0 = moe.moe_router_select(l[:0], 6)
    assert tuple(i0.shape) == (0, 6) and tuple(w0.shape) == (0, 6)


def test_refusals_without_gpu(moe):
    """Every one is refused before the first CUDA call."""
    L = moe.lib()
    p = 0x1000

    def call(logits=p, lt=0, ld=0, bias=None, ids=p, w=p, wt=1, T=4, E=16, K=2, G=1, topG=1, top=1, score=0, renorm=0):
        return L.MoeRouterSelect(logits, lt, ld, bias, ids, w, wt, T, E, K, G, topG, top, score, renorm, 1.0, None)

    for kw in (dict(T=-1), dict(E=0), dict(E=257), dict(K=0), dict(K=9), dict(K=17, E=16), dict(G=3), dict(G=0),
               dict(G=33, E=66), dict(G=4, topG=5), dict(G=4, topG=0), dict(G=8, topG=1, K=3), dict(top=0),
               dict(top=3), dict(G=16, topG=2, top=2), dict(ld=15), dict(ld=-1), dict(T=1 << 30, K=2)):
        assert call(**kw) == -2, kw
    for kw in (dict(lt=3), dict(lt=2), dict(wt=27), dict(wt=3), dict(score=2), dict(score=-1)):
        assert call(**kw) == -5, kw
    for kw in (dict(logits=None), dict(ids=None), dict(w=None)):
        assert call(**kw) == -1, kw
    for kw in (dict(logits=0x1002), dict(bias=0x1002), dict(ids=0x1002), dict(w=0x1001), dict(w=0x1002, wt=0)):
        assert call(**kw) == -6, kw
    assert call(T=0) == 0
    assert call(T=0, logits=None, ids=None, w=None) == 0


def test_front_end_refusals_without_gpu(moe):
    with pytest.raises(moe.MoeError):
        moe.moe_router_select(torch.zeros(2, 4), 2)  # no CPU fallback
    with pytest.raises(moe.MoeError):
        moe.moe_router_select([[1.0]], 1)


@pytest.mark.gpu
def test_front_end_refusals(moe, gpu):
    l = torch.zeros((4, 16), device="cuda")
    bad = [dict(logits=l.double()), dict(logits=l[0]), dict(logits=l.t()), dict(logits=l[:1].expand(4, 16)),
           dict(bias=torch.zeros(16)), dict(bias=torch.zeros(15, device="cuda")),
           dict(bias=torch.zeros(16, device="cuda", dtype=torch.float16)), dict(scoreFunc="tanh"), dict(topK=9),
           dict(numGroups=3), dict(expert_ids=torch.zeros((4, 2), dtype=torch.int64, device="cuda")),
           dict(expert_ids=torch.zeros((4, 3), dtype=torch.int32, device="cuda")),
           dict(weights=torch.zeros((4, 2), dtype=torch.bfloat16, device="cuda")),
           dict(weights=torch.zeros((4, 4), device="cuda")[:, :2]), dict(weights=torch.zeros((4, 2)))]
    for kw in bad:
        kw = dict(dict(logits=l, topK=2), **kw)
        with pytest.raises(moe.MoeError):
            moe.moe_router_select(**kw)
