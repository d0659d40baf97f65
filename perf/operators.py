"""Cases and plain forms of the routing and int8 operators.

Three operators:

  route    experts chosen from router logits (`route_experts`)
  linear   16-bit activations times an int8 weight matrix, tokens quantised on the fly (`int8_linear`)
  shared   the shared expert of an MoE layer: an int8 SwiGLU FFN that every token takes (`int8_shared_expert`)

With `own` false, `run` computes them from elementary torch operations; with
`own` true it makes the library's calls on the same state.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LARGEST_ROUTE = 32768 * 256          # logits of the largest routing case
LARGEST_LINEAR = 8192 * 7168 * 4096  # multiply-adds of the largest product
LARGEST_BYTES = 160 << 20            # activations of a drawn product
LARGEST_SHARED = 8192 * 7168 * 2048  # multiply-adds of one product of the largest shared expert


def _route(name, T, E, k, score, groups, kept, group_top, bias, renorm, scale, logits, pad=0, masked=0.0):
    return {"name": name, "op": "route", "T": T, "E": E, "k": k, "score": score, "groups": groups, "kept": kept,
            "group_top": group_top, "bias": bias, "renorm": renorm, "scale": scale, "logits": logits, "pad": pad,
            "masked": masked}


def _linear(name, T, K, N, x, out, order="kn", bias=False):
    return {"name": name, "op": "linear", "T": T, "K": K, "N": N, "x": x, "out": out, "order": order, "bias": bias}


def _shared(name, T, d, f, x, order="kn", residual=True):
    return {"name": name, "op": "shared", "T": T, "d": d, "f": f, "x": x, "order": order, "residual": residual}


def listed():
    return [
        # one decoded token at the 256-expert shape: launch latency
        _route("route_1x256", 1, 256, 8, "sigmoid", 8, 4, 2, True, True, 2.5, "f32"),
        # the 64-expert int8 workload's prefill, plain softmax gate, weights not renormalised
        _route("route_16384x64", 16384, 64, 6, "softmax", 1, 1, 1, False, False, 1.0, "bf16"),
        # the largest: prefill at 256 experts, sigmoid scores, balance bias, 4 of 8 groups
        _route("route_32768x256", 32768, 256, 8, "sigmoid", 8, 4, 2, True, True, 2.5, "f32"),
        # a ragged batch at 160 experts in groups of 20, logits a slice of a wider tensor, a fifth of them masked
        _route("route_1021x160_ragged", 1021, 160, 6, "softmax", 8, 3, 1, True, True, 16.0, "f16", pad=5, masked=0.2),
        # one decoded token through a 7168 x 2048 projection: weight bandwidth and latency
        _linear("linear_1x7168x2048", 1, 7168, 2048, "bf16", "bf16"),
        # a decode batch, wide output
        _linear("linear_512x2048x7168", 512, 2048, 7168, "bf16", "bf16"),
        # the largest: a prefill chunk
        _linear("linear_8192x7168x4096", 8192, 7168, 4096, "bf16", "bf16"),
        # odd sizes in each axis, [N, K] weights, bias, f32 result
        _linear("linear_333x1001x1407_odd", 333, 1001, 1407, "f16", "f32", order="nk", bias=True),
        # the shared expert of the 7168 / 2048 shape at one token
        _shared("shared_1x7168x2048", 1, 7168, 2048, "bf16"),
        # the same at the decode batch
        _shared("shared_512x7168x2048", 512, 7168, 2048, "bf16"),
        # the largest: the prefill batch
        _shared("shared_8192x7168x2048", 8192, 7168, 2048, "bf16"),
        # a ragged batch at an odd hidden size, f16, no residual
        _shared("shared_77x2048x1405_odd", 77, 2048, 1405, "f16", order="nk", residual=False),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], its logarithm spread evenly."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "linear", "shared"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        per = _log(rng, max(1, 8 // groups), 512 // groups)
        E = groups * per
        T = _log(rng, 1, min(32768, LARGEST_ROUTE // E))
        kept = rng.randint(1, groups)
        return {"op": op, "T": T, "E": E, "k": rng.randint(1, min(16, kept * per)), "score": rng.choice(["softmax", "sigmoid"]),
                "groups": groups, "kept": kept, "group_top": rng.choice([1, 2]), "bias": rng.random() < 0.6,
                "renorm": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5, 16.0]),
                "logits": rng.choice(["f32", "f32", "f16", "bf16"]), "pad": rng.choice([0, 0, 1, 8, 13]),
                "masked": rng.choice([0.0, 0.0, 0.1, 0.6])}
    if op == "linear":
        K, N = _log(rng, 32, 14336), _log(rng, 8, 14336)
        T = _log(rng, 1, max(1, min(16384, LARGEST_LINEAR // (K * N), LARGEST_BYTES // (2 * K + 4 * N))))
        if rng.random() < 0.5:
            K, N = max(16, K // 16 * 16), max(16, N // 16 * 16)
        return {"op": op, "T": T, "K": K, "N": N, "x": rng.choice(["bf16", "bf16", "f16"]),
                "out": rng.choice(["bf16", "f16", "f32"]), "order": rng.choice(["kn", "kn", "nk"]),
                "bias": rng.random() < 0.3}
    d, f = _log(rng, 64, 7168), _log(rng, 32, 8192)
    T = _log(rng, 1, max(1, min(16384, LARGEST_SHARED // (d * f), LARGEST_BYTES // (6 * d))))
    if rng.random() < 0.5:
        d, f = max(16, d // 16 * 16), max(16, f // 16 * 16)
    return {"op": op, "T": T, "d": d, "f": f, "x": rng.choice(["bf16", "bf16", "f16"]), "order": rng.choice(["kn", "kn", "nk"]),
            "residual": rng.random() < 0.5}


def _tokens(gen, T, K, dtype):
    """Activations: unit normal with a few channels an order of magnitude larger, as trained models have them."""
    x = torch.randn(T, K, generator=gen, device=DEV)
    loud = torch.randint(0, K, (max(1, K // 512),), generator=gen, device=DEV)
    x[:, loud] *= 12.0
    return x.to(dtype)


def _weight(gen, K, N, order):
    """An int8 matrix [K, N] with one f32 scale per column, quantised from N(0, 1/sqrt(K)); its rows (or, for "nk",
    its columns) start 16 bytes apart or a multiple of that."""
    w = torch.randn(K, N, generator=gen, device=DEV) * (1.0 / math.sqrt(K))
    scale = w.abs().amax(0) / 127.0
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    q = torch.clamp(torch.round(w / scale), -127, 127).to(torch.int8)
    if order == "kn":
        store = torch.zeros(K, (N + 15) // 16 * 16, dtype=torch.int8, device=DEV)
        store[:, :N] = q
        return store[:, :N], scale
    store = torch.zeros(N, (K + 15) // 16 * 16, dtype=torch.int8, device=DEV)
    store[:, :K] = q.t()
    return store[:, :K].t(), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(1000003 * seed + 17)
    c = dict(case)
    if c["op"] == "route":
        T, E = c["T"], c["E"]
        # logits of a trained router: a per-expert popularity, a per-token spread
        popular = 0.7 * torch.randn(E, generator=gen, device=DEV)
        x = 1.6 * torch.randn(T, E, generator=gen, device=DEV) + popular
        if c["masked"] > 0:
            hide = torch.rand(T, E, generator=gen, device=DEV) < c["masked"]
            x = torch.where(hide, torch.full_like(x, -math.inf), x)
            x[T // 3] = -math.inf   # one token that no expert may take
        store = torch.zeros(T, E + c["pad"], dtype=TYPES[c["logits"]], device=DEV)
        store[:, :E] = x.to(store.dtype)
        c["x"] = store[:, :E]
        c["b"] = 0.1 * torch.randn(E, generator=gen, device=DEV) if c["bias"] else None
    elif c["op"] == "linear":
        c["a"] = _tokens(gen, c["T"], c["K"], TYPES[c["x"]])
        c["w"], c["ws"] = _weight(gen, c["K"], c["N"], c["order"])
        c["b"] = torch.randn(c["N"], generator=gen, device=DEV) if c["bias"] else None
    else:
        T, d, f = c["T"], c["d"], c["f"]
        c["a"] = _tokens(gen, T, d, TYPES[c["x"]])
        c["wg"], c["sg"] = _weight(gen, d, f, c["order"])
        c["wu"], c["su"] = _weight(gen, d, f, c["order"])
        c["wd"], c["sd"] = _weight(gen, f, d, c["order"])
        c["r"] = torch.randn(T, d, generator=gen, device=DEV).to(TYPES[c["x"]]) if c["residual"] else None
    return c


# ---- plain forms ---------------------------------------------------------------


def _lowest(dtype):
    """Logits up to this value are masked."""
    return -65504.0 if dtype == torch.float16 else -1e20


def _route_plain(s):
    x, b = s["x"].double(), s["b"]
    T, E = x.shape
    G, k = s["groups"], s["k"]
    hidden = ~(x > _lowest(s["x"].dtype))
    x = torch.where(hidden, torch.full_like(x, -math.inf), x)
    if s["score"] == "sigmoid":
        logscore = torch.clamp(x, max=0.0) - torch.log1p(torch.exp(-x.abs()))
        score = 1.0 / (1.0 + torch.exp(-x))
    else:
        top = torch.clamp(x.amax(1, keepdim=True), min=-1e300)
        logscore = x - top
        e = torch.exp(logscore)
        score = e / torch.clamp(e.sum(1, keepdim=True), min=1e-300)
    # both scores grow with the logit: without a bias the logits give the order
    value = x if b is None else torch.where(hidden, x, score + b.double())
    if G > 1:
        member = value if s["group_top"] == 1 or b is not None else torch.where(hidden, x, score)
        best = member.reshape(T, G, E // G).sort(dim=2, descending=True).values
        of_group = best[:, :, 0]
        if s["group_top"] == 2 and E // G > 1:
            second = best[:, :, 1]
            of_group = of_group + torch.where(second == -math.inf, torch.zeros_like(second), second)
        order = of_group.sort(dim=1, descending=True, stable=True).indices[:, : s["kept"]]
        keep = torch.zeros(T, G, dtype=torch.bool, device=x.device)
        keep.scatter_(1, order, True)
        value = torch.where(keep.repeat_interleave(E // G, 1), value, torch.full_like(value, -math.inf))
    best, idx = value.sort(dim=1, descending=True, stable=True)
    best, idx = best[:, :k], idx[:, :k]
    none = best == -math.inf
    if s["renorm"]:
        chosen = torch.where(none, torch.full_like(best, -math.inf), logscore.gather(1, idx))
        e = torch.exp(chosen - torch.clamp(chosen.amax(1, keepdim=True), min=-1e300))
        w = e / torch.clamp(e.sum(1, keepdim=True), min=1e-300)
    else:
        w = score.gather(1, idx)
    w = torch.where(none, torch.zeros_like(w), w * s["scale"])
    return torch.where(none, torch.full_like(idx, -1), idx).int(), w.float()


def _quantize_plain(x):
    """Per-token symmetric int8: the quotient in 64 bits, so that values next to a rounding border fall on their side."""
    scale = x.float().abs().amax(1, keepdim=True) / 127.0
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    return torch.clamp(torch.round(x.double() / scale.double()), -127, 127).float(), scale


def _product_plain(q, scale, w, ws):
    return (q @ w.float()) * scale * ws


def _shared_plain(s):
    q, scale = _quantize_plain(s["a"])
    g = _product_plain(q, scale, s["wg"], s["sg"])
    u = _product_plain(q, scale, s["wu"], s["su"])
    hq, hs = _quantize_plain(u * (g / (1.0 + torch.exp(-g))))
    y = _product_plain(hq, hs, s["wd"], s["sd"])
    if s["r"] is not None:
        y = y + s["r"].float()
    return y.to(s["a"].dtype)


def run(state):
    s = state
    if own:
        import sparsemoe_b200 as sm
        if s["op"] == "route":
            return sm.route_experts(s["x"], s["k"], score=s["score"], bias=s["b"], groups=s["groups"],
                                    kept_groups=s["kept"], group_top=s["group_top"], renormalise=s["renorm"],
                                    scale=s["scale"])
        if s["op"] == "linear":
            return sm.int8_linear(s["a"], s["w"], s["ws"], bias=s["b"], out_dtype=TYPES[s["out"]])
        return sm.int8_shared_expert(s["a"], s["wg"], s["sg"], s["wu"], s["su"], s["wd"], s["sd"], residual=s["r"])
    if s["op"] == "route":
        return _route_plain(s)
    if s["op"] == "linear":
        q, scale = _quantize_plain(s["a"])
        y = _product_plain(q, scale, s["w"], s["ws"])
        if s["b"] is not None:
            y = y + s["b"]
        return y.to(TYPES[s["out"]])
    return _shared_plain(s)


def work(case):
    c = case
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if c["op"] == "route":
        n = c["T"] * c["E"]
        return {"bytes": n * size[c["logits"]] + 8 * c["T"] * c["k"] + (4 * c["E"] if c["bias"] else 0),
                "flops": 6 * n}
    if c["op"] == "linear":
        T, K, N = c["T"], c["K"], c["N"]
        return {"bytes": 2 * T * K + K * N + (8 if c["bias"] else 4) * N + T * N * size[c["out"]], "flops": 2 * T * K * N}
    T, d, f = c["T"], c["d"], c["f"]
    return {"bytes": 2 * T * d * (3 if c["residual"] else 2) + 3 * d * f + 4 * (2 * f + d), "flops": 6 * T * d * f}


# ---- from the definitions, in 64 bits -------------------------------------------


def _exact_route(s):
    """Row by row in numpy: scores, groups, the k first of the order, weights."""
    low = _lowest(s["x"].dtype)
    x = s["x"].double().cpu().numpy()
    T, E = x.shape
    b = None if s["b"] is None else s["b"].double().cpu().numpy()
    G, k, per = s["groups"], s["k"], E // s["groups"]
    with np.errstate(over="ignore"):
        seen = x > low
        if s["score"] == "sigmoid":
            p = np.where(seen, 1.0 / (1.0 + np.exp(-x)), 0.0)
        else:
            m = np.max(np.where(seen, x, -1e300), axis=1, keepdims=True)
            p = np.where(seen, np.exp(np.where(seen, x - m, 0.0)), 0.0)
            p = p / np.maximum(p.sum(1, keepdims=True), 1e-300)
    v = np.where(seen, x if b is None else p + b, -np.inf)
    if G > 1:
        t = np.where(seen, x if b is None and s["group_top"] == 1 else p if b is None else p + b, -np.inf)
        t = -np.sort(-t.reshape(T, G, per), axis=2)
        score = t[:, :, 0].copy()
        if s["group_top"] == 2 and per > 1:
            score += np.where(np.isfinite(t[:, :, 1]), t[:, :, 1], 0.0)
        rank = np.argsort(np.argsort(-score, axis=1, kind="stable"), axis=1, kind="stable")
        v = np.where(np.repeat(rank < s["kept"], per, axis=1), v, -np.inf)
    idx = np.argsort(-v, axis=1, kind="stable")[:, :k]
    empty = np.take_along_axis(v, idx, 1) == -np.inf
    w = np.where(empty, 0.0, np.take_along_axis(p, idx, 1))
    if s["renorm"]:
        w = w / np.maximum(w.sum(1, keepdims=True), 1e-300)
    return [torch.from_numpy(np.where(empty, -1, idx).astype(np.int32)), torch.from_numpy(w * s["scale"])]


def _exact_codes(x):
    s = x.abs().amax(1, keepdim=True) / 127.0
    s = torch.where(s > 0, s, torch.ones_like(s))
    return s, torch.round(x / s)


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "route":
        return _exact_route(s)
    x = s["a"].double()
    # the scales of the tokens are f32 numbers; the codes round the exact quotient
    sx, _ = _exact_codes(x)
    sx = sx.float().double()
    q = torch.round(x / sx)
    if s["op"] == "linear":
        y = torch.matmul(q, s["w"].double()) * (sx * s["ws"].double())
        return y if s["b"] is None else y + s["b"].double()
    g = torch.matmul(q, s["wg"].double()) * (sx * s["sg"].double())
    u = torch.matmul(q, s["wu"].double()) * (sx * s["su"].double())
    sh, qh = _exact_codes(torch.sigmoid(g) * g * u)
    y = torch.matmul(qh, s["wd"].double()) * (sh * s["sd"].double())
    return y if s["r"] is None else y + s["r"].double()
