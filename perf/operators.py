"""The cases that the router selection and the linear operator are measured on.

Two operators of an MoE layer, next to its routing, expert FFN and combine:

* ``router_select`` (``moe_router_select``): router logits [T, E] -> expert ids
  [T, K] and weights [T, K].  Scores are a softmax or a sigmoid of the logits; a
  per-expert bias may steer the choice but not the weight; experts may be chosen
  within the best few of several groups; weights may be renormalised and scaled.
* ``linear`` (``moe_linear``): y = act(x W^T + bias) + residual, or, gated,
  y = act(x Wg^T + bg) * (x Wu^T + bu) + residual: a router's gate, and the two
  projections of a shared expert.

``run`` computes them with elementary torch operations where ``own`` is false, and
with the library where it is true.
"""
import importlib

import numpy as np
import torch

own = False

_PACKAGE = "implementing-moe-architecture-operators-on-cann-platform_b200"
_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_NEG_INF = float("-inf")


def _router(T, E, K, dtype, score, G=1, topG=1, groupTop=1, bias=False, renorm=False, scale=1.0, out="float16",
            pad=0, masked=False):
    return {"op": "router_select", "T": T, "E": E, "K": K, "G": G, "topG": topG, "groupTop": groupTop,
            "dtype": dtype, "out": out, "score": score, "bias": bias, "renorm": renorm, "scale": scale,
            "pad": pad, "masked": masked}


def _linear(T, K, N, dtype, out=None, act="none", gated=False, bias=False, residual=False, pad=0):
    return {"op": "linear", "T": T, "K": K, "N": N, "dtype": dtype, "out": out or dtype, "act": act,
            "gated": gated, "bias": bias, "residual": residual, "pad": pad}


def listed():
    return [
        # One token of a large layer while it answers: latency is all that counts.  The
        # logits come in 32 bits from the gate; the balance bias steers the choice.
        {"name": "router_one_token",
         **_router(1, 256, 8, "float32", "sigmoid", 8, 4, 2, bias=True, renorm=True, scale=2.5)},
        # A decode batch of the 64-expert, 6-slot configuration, plain softmax scores.
        {"name": "router_decode", **_router(128, 64, 6, "float16", "softmax")},
        # Odd sizes, a padded row, groups of 15, one expert out of service in every row
        # and rows whose mask leaves few or none.
        {"name": "router_ragged",
         **_router(1337, 60, 4, "bfloat16", "softmax", 4, 2, 1, scale=1.5, out="float32", pad=4, masked=True)},
        # Prefill of the 64-expert configuration, softmax with a balance bias.
        {"name": "router_prefill", **_router(16384, 64, 6, "bfloat16", "softmax", bias=True, renorm=True)},
        # The largest: many prompts at once through a 256-expert router with groups.
        {"name": "router_large",
         **_router(65536, 256, 8, "float32", "sigmoid", 8, 4, 2, bias=True, renorm=True, scale=2.5)},
        # The router's gate for one token: logits in 32 bits.
        {"name": "gate_one_token", **_linear(1, 2048, 64, "float16", out="float32")},
        # A shared expert's down projection for a few sequences, added to the routed output.
        {"name": "down_few_tokens", **_linear(8, 8192, 2048, "float16", residual=True)},
        # A shared expert's gate and up projections for a decode batch.
        {"name": "gated_decode", **_linear(128, 2048, 8192, "float16", act="silu", gated=True)},
        # Odd sizes throughout, with padded rows, a bias, an activation and a residual.
        {"name": "linear_ragged",
         **_linear(777, 1416, 1411, "bfloat16", act="gelu", bias=True, residual=True, pad=8)},
        # The gate of a prefill batch: reads the activations once, writes a few columns.
        {"name": "gate_prefill", **_linear(16384, 2048, 64, "float16", out="float32")},
        # Prefill: a shared expert's down projection with a bias, added to the routed output.
        {"name": "down_prefill", **_linear(4096, 8192, 2048, "float16", bias=True, residual=True)},
        # The largest: gate and up projections of the 4096 x 14336 configuration.
        {"name": "gated_large", **_linear(8192, 4096, 14336, "bfloat16", act="silu", gated=True)},
    ]


def _log_int(rng, lo, hi):
    return int(round(np.exp(rng.uniform(np.log(lo), np.log(hi)))))


def draw(rng):
    if rng.random() < 0.45:
        T = _log_int(rng, 1, 65536)
        E = rng.choice([rng.randint(2, 256), 8, 16, 60, 64, 128, 160, 256])
        G = rng.choice([g for g in range(1, 33) if E % g == 0]) if rng.random() < 0.6 else 1
        groupTop = rng.choice([1, 2]) if E // G >= 2 else 1
        topG = rng.randint(1, G)
        K = rng.randint(1, min(8, topG * (E // G)))
        return _router(T, E, K, rng.choice(sorted(_TYPES)), rng.choice(["softmax", "sigmoid"]), G, topG, groupTop,
                       bias=rng.random() < 0.6, renorm=rng.random() < 0.6, scale=rng.choice([1.0, 1.5, 2.5]),
                       out=rng.choice(["float16", "float32"]), pad=rng.choice([0, 0, 1, 8]),
                       masked=rng.random() < 0.25)
    while True:
        T, K, N = _log_int(rng, 1, 16384), 8 * _log_int(rng, 4, 1792), _log_int(rng, 1, 16384)
        gated = rng.random() < 0.4
        if 2.0 * T * K * N * (2 if gated else 1) <= 1.9e12:
            break
    dtype = rng.choice(["float16", "bfloat16"])
    return _linear(T, K, N, dtype, out=rng.choice([dtype, dtype, "float32"]),
                   act=rng.choice(["none", "relu", "gelu", "gelu_tanh", "silu", "sigmoid"]), gated=gated,
                   bias=rng.random() < 0.5, residual=rng.random() < 0.5, pad=rng.choice([0, 0, 8, 24]))


def _padded(t, pad):
    """t with `pad` more elements between the end of one row and the start of the next."""
    if not pad:
        return t
    wide = torch.zeros((t.shape[0], t.shape[1] + pad), dtype=t.dtype, device=t.device)
    wide[:, :t.shape[1]] = t
    return wide[:, :t.shape[1]]


def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1_000_003 * seed + 17)

    def normal(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)

    dt = _TYPES[case["dtype"]]
    s = {}
    if case["op"] == "router_select":
        T, E = case["T"], case["E"]
        # what a gate gives: a spread of about one per token, some experts liked more than others
        logits = normal(T, E) * 1.3 + normal(E) * 0.4
        if case["masked"]:
            logits[:, E // 3] = _NEG_INF                          # out of service
            rows = torch.rand((T, 1), generator=g, device="cuda")  # a few rows keep little or nothing
            keep = torch.rand((T, E), generator=g, device="cuda") < 2.0 / E
            logits = torch.where((rows < 0.05) & ~keep, _NEG_INF, logits)
        s["logits"] = _padded(logits.to(dt), case["pad"])
        # the balance bias moves in fixed small steps, so experts share values
        s["bias"] = torch.round(normal(E) * 30.0) * 0.001 if case["bias"] else None
        return s
    T, K, N = case["T"], case["K"], case["N"]
    rows = 2 * N if case["gated"] else N
    s["x"] = _padded(normal(T, K).to(dt), case["pad"])
    s["weight"] = (normal(rows, K) / K ** 0.5).to(dt)
    s["bias"] = (normal(rows) * 0.2).to(dt) if case["bias"] else None
    s["residual"] = _padded(normal(T, N).to(_TYPES[case["out"]]), case["pad"]) if case["residual"] else None
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    out = _TYPES[case["out"]]
    if own:
        s["moe"] = importlib.import_module(_PACKAGE)
        if case["op"] == "router_select":
            s["ids"] = torch.empty((case["T"], case["K"]), dtype=torch.int32, device="cuda")
            s["weights"] = torch.empty((case["T"], case["K"]), dtype=out, device="cuda")
        else:
            s["y"] = torch.empty((case["T"], case["N"]), dtype=out, device="cuda")
    return s


def run(state):
    c = state["case"]
    if own:
        moe = state["moe"]
        if c["op"] == "router_select":
            return moe.moe_router_select(state["logits"], c["K"], bias=state["bias"], numGroups=c["G"],
                                         topGroups=c["topG"], groupTop=c["groupTop"], scoreFunc=c["score"],
                                         renormalize=c["renorm"], scale=c["scale"], expert_ids=state["ids"],
                                         weights=state["weights"])
        return moe.moe_linear(state["x"], state["weight"], bias=state["bias"], activation=c["act"],
                              gated=c["gated"], residual=state["residual"], y=state["y"])
    return _plain_router(state, c) if c["op"] == "router_select" else _plain_linear(state, c)


def _plain_router(s, c):
    """Scores in 64 bits: the choice hangs on scores next to one another."""
    T, E, K, G = c["T"], c["E"], c["K"], c["G"]
    x = s["logits"].double()
    open_ = x != _NEG_INF
    if c["score"] == "softmax":
        top = x.amax(1, keepdim=True)
        e = torch.exp(x - torch.where(torch.isinf(top), 0.0, top))
        score = e / e.sum(1, keepdim=True).clamp_min(1e-300)
    else:
        score = 1.0 / (1.0 + torch.exp(-x))
    key = score if s["bias"] is None else score + s["bias"].double()
    key = torch.where(open_, key, _NEG_INF)
    if G > 1:
        best = key.view(T, G, E // G).sort(dim=2, descending=True).values[:, :, :c["groupTop"]]
        some = best[:, :, 0] != _NEG_INF
        group = torch.where(best == _NEG_INF, 0.0, best).sum(2)
        group = torch.where(some, group, _NEG_INF)
        order = group.sort(dim=1, descending=True, stable=True).indices[:, :c["topG"]]
        chosen = torch.zeros((T, G), dtype=torch.bool, device=x.device).scatter_(1, order, True)
        key = torch.where(chosen.repeat_interleave(E // G, 1), key, _NEG_INF)
    ids = key.sort(dim=1, descending=True, stable=True).indices[:, :K]
    w = torch.where(key.gather(1, ids) == _NEG_INF, 0.0, score.gather(1, ids))
    if c["renorm"]:
        w = w / w.sum(1, keepdim=True).clamp_min(1e-300)
    return ids.int(), (w * c["scale"]).to(_TYPES[c["out"]])


def _plain_act(z, name):
    if name == "relu":
        return torch.where(z > 0, z, 0.0)
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * 0.5 ** 0.5))
    if name == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh((2.0 / np.pi) ** 0.5 * (z + 0.044715 * z * z * z)))
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "sigmoid":
        return 1.0 / (1.0 + torch.exp(-z))
    return z


def _plain_linear(s, c):
    z = s["x"].float() @ s["weight"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _plain_act(z[:, :c["N"]], c["act"]) * z[:, c["N"]:] if c["gated"] else _plain_act(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(_TYPES[c["out"]])


def work(case):
    size = {"float32": 4, "float16": 2, "bfloat16": 2}
    T = case["T"]
    if case["op"] == "router_select":
        E, K = case["E"], case["K"]
        # per expert an exponential, a division, a bias and K comparisons
        return {"bytes": T * E * size[case["dtype"]] + T * K * (4 + size[case["out"]]) + (E * 4 if case["bias"] else 0),
                "flops": T * E * (4 + K)}
    K, N = case["K"], case["N"]
    rows = 2 * N if case["gated"] else N
    b = (T * K + rows * K) * size[case["dtype"]] + T * N * size[case["out"]]
    b += rows * size[case["dtype"]] if case["bias"] else 0
    b += T * N * size[case["out"]] if case["residual"] else 0
    return {"bytes": b, "flops": 2 * T * K * rows}


def exact(case, seed):
    s = _inputs(case, seed)
    return _exact_router(case, s) if case["op"] == "router_select" else _exact_linear(case, s)


def _exact_router(c, s):
    """Row by row over sorted keys, in numpy's 64 bits."""
    x = s["logits"].cpu().double().numpy()
    T, E = x.shape
    G, size = c["G"], E // c["G"]
    open_ = x > _NEG_INF
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if c["score"] == "softmax":
            low = np.where(open_, x, -np.inf).max(axis=1, initial=-np.inf)
            low[~np.isfinite(low)] = 0.0
            score = np.exp(x - low[:, None])
            total = score.sum(axis=1)
            total[total == 0.0] = 1.0
            score /= total[:, None]
        else:
            score = np.reciprocal(1.0 + np.exp(-x))
    steer = score.copy()
    if s["bias"] is not None:
        steer += s["bias"].cpu().numpy().astype(np.float64)[None, :]
    steer[~open_] = -np.inf
    if G > 1:
        blocks = np.sort(steer.reshape(T, G, size), axis=2)
        value = blocks[:, :, -1].copy()
        if c["groupTop"] == 2:
            second = blocks[:, :, -2]
            value += np.where(np.isinf(second), 0.0, second)
        rank = np.argsort(np.argsort(-value, axis=1, kind="stable"), axis=1, kind="stable")
        steer[np.repeat(rank >= c["topG"], size, axis=1)] = -np.inf
    ids = np.argsort(-steer, axis=1, kind="stable")[:, :c["K"]]
    w = np.take_along_axis(score, ids, 1)
    w[np.isinf(np.take_along_axis(steer, ids, 1))] = 0.0
    if c["renorm"]:
        total = w.sum(axis=1, keepdims=True)
        w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
    return (torch.from_numpy(ids.astype(np.int32)).cuda(), torch.from_numpy(w * c["scale"]).cuda())


def _exact_linear(c, s):
    """In 64 bits, a block of output columns at a time."""
    x = s["x"].double()
    N = c["N"]
    y = torch.empty((c["T"], N), dtype=torch.float64, device="cuda")
    for lo in range(0, N, 4096):
        hi = min(lo + 4096, N)

        def part(first):
            z = torch.mm(x, s["weight"][first + lo:first + hi].double().t())
            return z if s["bias"] is None else z.add_(s["bias"][first + lo:first + hi].double())

        z = part(0)
        a = {"none": lambda: z, "relu": lambda: z.clamp_min(0.0),
             "gelu": lambda: z * 0.5 * torch.special.erfc(-z / 2.0 ** 0.5),
             "gelu_tanh": lambda: z * torch.sigmoid(2.0 * (2.0 / np.pi) ** 0.5 * (z + 0.044715 * z ** 3)),
             "silu": lambda: z * torch.sigmoid(z), "sigmoid": lambda: torch.sigmoid(z)}[c["act"]]()
        y[:, lo:hi] = a * part(N) if c["gated"] else a
    if s["residual"] is not None:
        y += s["residual"].double()
    return y
