"""Plain 64-bit restatements of the stand-alone operators, for their tests."""
import numpy as np
import torch

LOWEST = {torch.float32: -1e20, torch.bfloat16: -1e20, torch.float16: -65504.0}


def route_ref(logits, k, score, bias, groups, kept, group_top, renorm, scale):
    """Row by row, from the definition.  Returns (indices, weights f64)."""
    low = LOWEST[logits.dtype]
    x = logits.double().cpu().numpy()
    b = None if bias is None else bias.double().cpu().numpy()
    T, E = x.shape
    per = E // groups
    idx, wts = np.full((T, k), -1, np.int64), np.zeros((T, k))
    with np.errstate(all="ignore"):
        for t in range(T):
            seen = [e for e in range(E) if x[t, e] > low and (b is None or b[e] > -1e20)]
            visible = [e for e in range(E) if x[t, e] > low]      # the softmax runs over these
            s = np.zeros(E)
            if score == "sigmoid":
                s[visible] = 1.0 / (1.0 + np.exp(-x[t, visible]))
            elif visible:
                m = max(x[t, e] for e in visible)
                ex = {e: 1.0 if x[t, e] == m else float(np.exp(x[t, e] - m)) for e in visible}
                for e in visible:
                    s[e] = ex[e] / sum(ex.values())
            value = {e: x[t, e] if b is None else s[e] + b[e] for e in seen}
            if groups > 1:
                marks = {}
                for g in range(groups):
                    mem = [e for e in seen if e // per == g]
                    if not mem:
                        continue
                    v = sorted((value[e] if b is not None or group_top == 1 else s[e] for e in mem), reverse=True)
                    marks[g] = sum(v[:group_top])
                # sums of two that agree to 2^-49 are ties (sigmoid(x) + sigmoid(-x) is 1 for every x)
                tie, stay = 2.0 ** -49 if group_top == 2 else 0.0, []
                while marks and len(stay) < kept:
                    m = max(marks.values())
                    g = min(g for g in marks if marks[g] >= (m if np.isinf(m) else m - tie * (1 + abs(m))))
                    stay.append(g)
                    del marks[g]
                value = {e: v for e, v in value.items() if e // per in stay}
            chosen = sorted(value, key=lambda e: (-value[e], e))[:k]
            if not chosen:
                continue
            w = np.array([s[e] for e in chosen])
            if renorm:
                xs = np.array([x[t, e] for e in chosen])
                ls = xs if score == "softmax" else np.minimum(xs, 0.0) - np.log1p(np.exp(-np.abs(xs)))
                w = np.where(ls == ls.max(), 1.0, np.exp(ls - ls.max()))
                w = w / w.sum()
            idx[t, : len(chosen)] = chosen
            wts[t, : len(chosen)] = w * scale
    return idx, wts


def quantize_ref(x):
    """(codes, scale) of the rows of x: scale f32, codes of the exact quotient (f64 holds it far from any tie it is not)."""
    x = x.detach().cpu()
    amax = x.float().abs().amax(1)
    s = (amax.numpy() * (np.float32(1.0) / np.float32(127.0))).astype(np.float32)
    s = np.where(s == 0, np.float32(1.0), s)
    q = np.rint(x.double().numpy() / s.astype(np.float64)[:, None])
    return np.clip(q, -127, 127), s


def matmul_ref(q, s, w, ws, bias=None):
    """f64 product, and the sum of magnitudes that its f32 roundings scale with."""
    y = (q @ w.double().cpu().numpy()) * s.astype(np.float64)[:, None] * ws.double().cpu().numpy()
    mag = np.abs(y)
    if bias is not None:
        y = y + bias.double().cpu().numpy()
        mag = mag + np.abs(bias.double().cpu().numpy())
    return y, mag


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """Half of the smallest subnormal: the rounding error near zero."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def int8_matrix(gen, K, N, order, device):
    """Random int8 weights [K, N] (every code, -128 too) with padded rows, and positive scales."""
    q = torch.randint(-128, 128, (K, N), generator=gen, dtype=torch.int8)
    if order == "kn":
        store = torch.full((K, (N + 15) // 16 * 16), 77, dtype=torch.int8)
        store[:, :N] = q
        w = store.to(device)[:, :N]
    else:
        store = torch.full((N, (K + 15) // 16 * 16), 77, dtype=torch.int8)
        store[:, :K] = q.t()
        w = store.to(device)[:, :K].t()
    ws = torch.rand(N, generator=gen) * 0.01 + 0.001
    return w, ws.to(device)
