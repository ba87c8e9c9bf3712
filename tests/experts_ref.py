"""The expert operators from their definitions in 64 bits on the CPU, point by point."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F32_MAX = torch.finfo(torch.float32).max


def route(scores, top_k, score_func="softmax", bias=None, n_groups=1, top_groups=None, renormalize=True, scale=1.0):
    """(weights float64 [N, k], indices [N, k]) as Python computes them, one row at a time."""
    top_groups = n_groups if top_groups is None else top_groups
    N, K = scores.shape
    per = K // n_groups
    weights, indices = torch.zeros(N, top_k, dtype=torch.float64), torch.full((N, top_k), -1, dtype=torch.int32)
    for n, row in enumerate(scores.double().tolist()):
        z = [min(v, F32_MAX) if v > -math.inf else None for v in row]
        live = [e for e in range(K) if z[e] is not None]
        if not live:
            continue
        m = max(z[e] for e in live)
        if score_func == "softmax":
            total = sum(math.exp(z[e] - m) for e in live)
            s = {e: math.exp(z[e] - m) / total for e in live}
        elif score_func == "sigmoid":
            s = {e: 1.0 / (1.0 + math.exp(-z[e])) if z[e] > -700 else math.exp(max(z[e], -745.0)) for e in live}
        else:
            s = {e: z[e] for e in live}
        if bias is None and top_groups == n_groups:
            c = {e: z[e] for e in live}
        else:
            c = {e: s[e] + (0.0 if bias is None else float(bias[e])) for e in live}
        c = {e: v for e, v in c.items() if v > -math.inf}
        if top_groups < n_groups:
            sums = {}
            for g in range(n_groups):
                best = sorted((c[e] for e in c if e // per == g), reverse=True)[:2]
                if best:
                    sums[g] = sum(best)
            kept = sorted(sums, key=lambda g: (-sums[g], g))[:top_groups]
            c = {e: v for e, v in c.items() if e // per in kept}
        chosen = sorted(c, key=lambda e: (-c[e], e))[:top_k]
        if not chosen:
            continue
        w = [s[e] for e in chosen]
        if renormalize:
            if score_func == "softmax":  # the same ratios without underflow
                mc = max(z[e] for e in chosen)
                w = [math.exp(z[e] - mc) for e in chosen]
            w = [v / sum(w) for v in w] if sum(w) != 0 else [0.0] * len(w)
        for j, e in enumerate(chosen):
            weights[n, j], indices[n, j] = scale * w[j], e
    return weights, indices


def weights_of(z, indices, score_func, renormalize, scale):
    """The weights as a differentiable float64 function of the scores, for given indices."""
    live = indices >= 0
    at = indices.long().clamp(min=0)
    zm = torch.where(torch.isnan(z), torch.full_like(z, -math.inf), z)
    if score_func == "softmax":
        s = torch.softmax(zm, 1)
    elif score_func == "sigmoid":
        s = torch.sigmoid(zm)
    else:
        s = zm
    w = torch.where(live, s.gather(1, at), torch.zeros((), dtype=z.dtype))
    if renormalize:
        w = w / w.sum(1, keepdim=True)
    return scale * w


def group(indices, K):
    flat = indices.reshape(-1).tolist()
    lists = [[i for i, e in enumerate(flat) if e == k] for k in range(K)]
    lost = [i for i, e in enumerate(flat) if not 0 <= e < K]
    offsets = [0]
    for a in lists:
        offsets.append(offsets[-1] + len(a))
    order = [i for a in lists for i in a] + lost
    position = [-1] * len(flat)
    for r, i in enumerate(order[:offsets[-1]]):
        position[i] = r
    return (torch.tensor(order, dtype=torch.int32), torch.tensor(offsets, dtype=torch.int32),
            torch.tensor(position, dtype=torch.int32).reshape(indices.shape))


def products(x, weight, order, offsets, top_k, dy=None):
    """y, and with dy also dx and dweight; float64 results and the sums of the products' magnitudes."""
    x, weight = x.double(), weight.double()
    R, (K, d_out, d_in) = order.numel(), weight.shape
    y, ya = (torch.zeros(R, d_out, dtype=torch.float64, device=x.device) for _ in range(2))
    dx, dxa = torch.zeros_like(x), torch.zeros_like(x)
    dw, dwa = torch.zeros_like(weight), torch.zeros_like(weight)
    off = offsets.tolist()
    for e in range(K):
        rows = slice(off[e], off[e + 1])
        n = order[rows].long() // top_k
        if n.numel() == 0:
            continue
        y[rows] = x[n] @ weight[e].T
        ya[rows] = x[n].abs() @ weight[e].abs().T
        if dy is not None:
            g = dy[rows].double()
            dw[e], dwa[e] = g.T @ x[n], g.abs().T @ x[n].abs()
            dx.index_add_(0, n, g @ weight[e])
            dxa.index_add_(0, n, g.abs() @ weight[e].abs())
    return (y, ya) if dy is None else (y, ya, dx, dxa, dw, dwa)


def combine(y, weights, position, d_out=None):
    y, weights = y.double(), weights.double()
    N, k = position.shape
    out, out_abs = torch.zeros(N, y.shape[1]).double(), torch.zeros(N, y.shape[1]).double()
    dy, dw = torch.zeros_like(y), torch.zeros(N, k).double()
    dwa = torch.zeros(N, k).double()
    for n in range(N):
        for j in range(k):
            p = int(position[n, j])
            if p < 0:
                continue
            out[n] += weights[n, j] * y[p]
            out_abs[n] += (weights[n, j] * y[p]).abs()
            if d_out is not None:
                g = d_out[n].double()
                dy[p] = weights[n, j] * g
                dw[n, j], dwa[n, j] = (g * y[p]).sum(), (g * y[p]).abs().sum()
    return (out, out_abs) if d_out is None else (out, out_abs, dy, dw, dwa)
