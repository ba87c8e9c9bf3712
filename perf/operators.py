"""What is measured of the expert operators: routing a score matrix to its top experts, grouping
the routes by expert, the experts' products over the grouped rows, and the weighted join of their
results, each forward and, where a model learns through it, backward.

``own = False`` computes them in elementary torch operations, ``own = True`` through
``flashgmm_b200.flash_gmm_native``.  ``listed()`` gives the named cases, ``draw(rng)`` more of the
same ranges, ``prepare(case, seed)`` a case's inputs, ``run(state)`` one pass, ``work(case)`` the
bytes and operations that it cannot do without, and ``exact(case, seed)`` its result in 64 bits.
"""
import numpy as np
import torch

own = False

DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


# ----------------------------------------------------------------------------- the cases
def _route(name, op, N, K, k, dtype, func, bias, n_groups, top_groups, renormalize, scale, padded):
    return {"name": name, "op": op, "N": N, "K": K, "top_k": k, "dtype": dtype, "score_func": func, "bias": bias,
            "n_groups": n_groups, "top_groups": top_groups, "renormalize": renormalize, "scale": scale, "padded": padded}


def _group(name, N, K, k, padded):
    return {"name": name, "op": "group", "N": N, "K": K, "top_k": k, "padded": padded}


def _products(name, op, N, K, k, d_in, d_out, dtype, padded):
    return {"name": name, "op": op, "N": N, "K": K, "top_k": k, "d_in": d_in, "d_out": d_out, "dtype": dtype, "padded": padded}


def _combine(name, op, N, K, k, d, dtype, padded):
    return {"name": name, "op": op, "N": N, "K": K, "top_k": k, "d_out": d, "dtype": dtype, "padded": padded}


def listed():
    return [
        # one new token of a serving loop: 256 experts in 8 groups, a balance bias on the selection
        _route("route one token", "route", 1, 256, 8, "float32", "sigmoid", True, 8, 4, True, 2.5, False),
        # a prompt batch through the same router, scores straight from a bf16 projection, some rows padding
        _route("route prompt", "route", 16384, 256, 8, "bfloat16", "sigmoid", True, 8, 4, True, 2.5, True),
        # the leading components of every point from an E-step's responsibilities (N and K of the larger fits)
        _route("route responsibilities", "route", 65536, 1024, 8, "float32", "given", False, 1, 1, True, 1.0, False),
        # a training step of a softmax router: the weights and the scores' gradient, an odd number of points
        _route("route train", "route_train", 65521, 128, 2, "float32", "softmax", False, 1, 1, False, 1.0, False),
        # the routes of a small decoding batch
        _group("group few", 37, 64, 4, True),
        # the routes of a whole data set over many components
        _group("group many", 65536, 1024, 8, False),
        # sixteen tokens decoded together: each expert that is met has a few rows, its weights are read once
        _products("products decode", "products", 16, 64, 4, 1024, 2048, "bfloat16", False),
        # a prompt batch through the experts
        _products("products prompt", "products", 8192, 64, 4, 1024, 2048, "bfloat16", True),
        # a training step with ragged sizes: products, and the gradients of inputs and weights
        _products("products train", "products_train", 4093, 16, 2, 1000, 1016, "float16", False),
        # linear experts behind the mixture's own sizes (256 components, 128 dimensions), in its own type
        _products("products train fp32", "products_train", 65536, 256, 2, 128, 128, "float32", False),
        # the join after a prompt batch
        _combine("combine prompt", "combine", 8192, 64, 4, 2048, "bfloat16", True),
        # the join of a training step and its gradients, in the mixture's own type
        _combine("combine train", "combine_train", 16411, 16, 2, 1000, "float32", False),
    ]


def _between(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return int(min(high, max(low, round(low * (high / low) ** rng.random()))))


def _unnamed(case):
    return {q: v for q, v in case.items() if q != "name"}


def draw(rng):
    op = rng.choice(["route", "route", "route_train", "group", "products", "products", "products_train", "combine", "combine_train"])
    padded = rng.random() < 0.4
    if op in ("route", "route_train"):
        while True:
            N, K = _between(rng, 1, 65536), _between(rng, 4, 1024)
            n_groups = rng.choice([1, 1, 2, 4, 8])
            K = max(n_groups * 2, K // n_groups * n_groups)
            if N * K <= 65536 * 1024:
                break
        top_groups = rng.randint(1, n_groups)
        k = rng.randint(1, min(8, K // n_groups * top_groups))
        func = rng.choice(["softmax", "sigmoid", "given"])
        return _unnamed(_route("", op, N, K, k, rng.choice(sorted(DTYPES)), func, rng.random() < 0.5, n_groups, top_groups,
                               rng.random() < 0.6, rng.choice([1.0, 2.5]), padded))
    if op == "group":
        N, K, k = _between(rng, 1, 65536), _between(rng, 4, 1024), rng.randint(1, 8)
        k = min(k, K)
        return _unnamed(_group("", N, K, k, padded))
    if op in ("products", "products_train"):
        while True:
            N, K, k = _between(rng, 1, 16384), _between(rng, 4, 256), rng.randint(1, 4)
            step = rng.choice([1, 8, 64])
            d_in, d_out = (max(step, _between(rng, 16, 2048) // step * step) for _ in range(2))
            if N * k * d_in * d_out * (3 if op == "products_train" else 1) <= 8192 * 4 * 1024 * 2048 and K * d_in * d_out <= 64 * 1024 * 2048:
                break
        k = min(k, K)
        return _unnamed(_products("", op, N, K, k, d_in, d_out, rng.choice(sorted(DTYPES)), padded))
    while True:
        N, K, k, d = _between(rng, 1, 65536), _between(rng, 4, 256), rng.randint(1, 8), _between(rng, 8, 4096)
        if N * k * d <= 8192 * 4 * 2048:
            break
    k = min(k, K)
    return _unnamed(_combine("", op, N, K, k, d, rng.choice(sorted(DTYPES)), padded))


# ---------------------------------------------------------------------------- the inputs
def _routes(indices, K):
    """The plan that a user's program keeps between the operators: the routes sorted by expert (those
    without one last), where each expert's begin, and the grouped row of each route (-1: none)."""
    flat = indices.reshape(-1).long()
    order = torch.sort(torch.where(flat < 0, K, flat), stable=True)[1]
    offsets = torch.zeros(K + 1, dtype=torch.int64, device=flat.device)
    offsets[1:] = torch.bincount(flat[flat >= 0], minlength=K).cumsum(0)
    position = torch.empty_like(flat)
    position[order] = torch.arange(flat.numel(), device=flat.device)
    position[flat < 0] = -1
    return order.int(), offsets.int(), position.int().reshape(indices.shape)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    N, K, k, op = case["N"], case["K"], case["top_k"], case["op"]
    state = {"case": case}
    if op in ("route", "route_train"):
        z = randn(N, K) * 1.5 + randn(K) * 0.5
        if case["score_func"] == "given":  # responsibilities: a few components hold a point's mass
            z = torch.softmax(4.0 * z, dim=1)
        if case["padded"]:  # the last rows of a padded batch route nowhere; a few experts are switched off
            z[N - N // 8:] = -float("inf")
            z[:, 3::64] = -float("inf")
        state["scores"] = z.to(DTYPES[case["dtype"]])
        state["bias"] = randn(K) * 0.05 if case["bias"] else None
        if op == "route_train":
            state["d_weights"] = randn(N, k)
        return state
    # experts differ in popularity: the most wanted get several times the mean
    wanted = randn(N, K) + randn(K) * 0.5
    indices = torch.topk(wanted, k, dim=1)[1].int()
    if case["padded"]:
        indices[N - N // 8:] = -1
    state["indices"] = indices
    if op == "group":
        return state
    state["order"], state["offsets"], state["position"] = _routes(indices, K)
    dtype, R, d_out = DTYPES[case["dtype"]], N * k, case["d_out"]
    if op in ("products", "products_train"):
        d_in = case["d_in"]
        state["x"] = randn(N, d_in).to(dtype)
        state["weight"] = (randn(K, d_out, d_in) / d_in ** 0.5).to(dtype)
        if op == "products_train":
            state["dy"] = randn(R, d_out).to(dtype)
        return state
    state["y"] = randn(R, d_out).to(dtype)
    w = torch.softmax(randn(N, k), dim=1)
    state["weights"] = torch.where(indices >= 0, w, torch.zeros_like(w))
    if op == "combine_train":
        state["d_out"] = randn(N, d_out).to(dtype)
    return state


# ------------------------------------------------------------------------ the plain forms
def _choose(z, bias, func, n_groups, top_groups, k):
    """Chosen experts, best first, ties to the lowest index; -1 where none is left.  Compared in
    64 bits: neighbours on the border of the top k differ by less than 32 bits resolve."""
    N, K = z.shape
    z = z.double()
    dead = torch.isnan(z) | (z == -float("inf"))
    z = z.clamp(max=torch.finfo(torch.float32).max)
    if bias is None and n_groups == 1:
        c = z
    else:
        if func == "softmax":
            e = torch.exp(z - torch.where(dead, -float("inf"), z).amax(1, keepdim=True))
            e = torch.where(dead, 0.0, e)
            c = e / e.sum(1, keepdim=True)
        else:
            c = 1.0 / (1.0 + torch.exp(-z)) if func == "sigmoid" else z
        if bias is not None:
            c = c + bias.double()
    c = torch.where(dead, -float("inf"), c)
    if n_groups > 1:
        best = torch.sort(c.view(N, n_groups, K // n_groups), dim=2, descending=True)[0][:, :, :2]
        none = best[:, :, 0] == -float("inf")
        score = torch.where(none, -float("inf"), torch.where(best == -float("inf"), 0.0, best).sum(2))
        kept = torch.sort(score, dim=1, descending=True, stable=True)[1][:, :top_groups]
        keep = torch.zeros_like(score, dtype=torch.bool).scatter(1, kept, True)
        c = torch.where(keep.repeat_interleave(K // n_groups, dim=1), c, -float("inf"))
    top, idx = torch.sort(c, dim=1, descending=True, stable=True)
    return torch.where(top[:, :k] == -float("inf"), -1, idx[:, :k])


def _shares(z, func, chosen):
    """The chosen scores' shares of their sum, from the scores (a ratio of two that both underflow
    is still their ratio), and the shares' sum before the division."""
    live = chosen >= 0
    zc = torch.gather(z, 1, chosen.clamp(min=0))
    if func == "given":
        t = torch.where(live, zc, 0.0)
        total = t.sum(1, keepdim=True)
        return torch.where(total == 0, 0.0, t / total), total
    top = torch.where(live, zc, -float("inf")).amax(1, keepdim=True)
    top = torch.where(top == -float("inf"), 0.0, top)
    if func == "softmax":
        t = torch.where(live, torch.exp(zc - top), 0.0)
    else:
        t = torch.where(live, torch.exp(zc.clamp(max=0) - top.clamp(max=0)) / (1.0 + torch.exp(-zc.abs())), 0.0)
    total = t.sum(1, keepdim=True)
    return torch.where(total == 0, 0.0, t / total), total


def _softmax(z):
    dead = torch.isnan(z) | (z == -float("inf"))
    top = torch.where(dead, -float("inf"), z).amax(1, keepdim=True)
    e = torch.where(dead, 0.0, torch.exp(z - torch.where(top == -float("inf"), 0.0, top)))
    total = e.sum(1, keepdim=True)
    return torch.where(total == 0, 0.0, e / total)


def _route_plain(s, case):
    func, k, scale = case["score_func"], case["top_k"], case["scale"]
    chosen = _choose(s["scores"], s["bias"], func, case["n_groups"], case["top_groups"], k)
    z = s["scores"].float().clamp(max=torch.finfo(torch.float32).max)
    live, at = chosen >= 0, chosen.clamp(min=0)
    if case["renormalize"]:
        w = _shares(z, func, chosen)[0]
    else:
        values = _softmax(z) if func == "softmax" else torch.sigmoid(z) if func == "sigmoid" else z
        w = torch.where(live, torch.gather(values, 1, at), 0.0)
    w = w * scale
    if case["op"] == "route":
        return [w, chosen.int()]
    g = torch.where(live, s["d_weights"] * scale, 0.0)
    dz = torch.zeros_like(z)
    if case["renormalize"]:
        p, total = _shares(z, func, chosen)
        dzc = g - (p * g).sum(1, keepdim=True)
        if func == "given":
            dzc = torch.where(total == 0, 0.0, dzc / total)
        else:
            dzc = p * dzc
            if func == "sigmoid":
                dzc = dzc * torch.sigmoid(-torch.gather(z, 1, at))
    else:
        zc = torch.gather(z, 1, at)
        if func == "softmax":
            v = torch.gather(values, 1, at)
            dz = -values * torch.where(live, v * g, 0.0).sum(1, keepdim=True)
            dzc = v * g
        elif func == "sigmoid":
            dzc = g * torch.sigmoid(zc) * torch.sigmoid(-zc)
        else:
            dzc = g
    dz = dz.scatter_add(1, at, torch.where(live, dzc, 0.0))
    return [w, chosen.int(), dz.to(s["scores"].dtype)]


def _padded(s, K):
    """Each expert's rows in a block of equal size: the place of every grouped row, and the blocks' length."""
    offsets = s["offsets"].long()
    counts = offsets[1:] - offsets[:-1]
    n, cap = int(offsets[-1]), max(1, int(counts.max()))
    expert = torch.repeat_interleave(torch.arange(K, device=counts.device), counts, output_size=n)
    return expert * cap + torch.arange(n, device=counts.device) - offsets[expert], n, cap


def _products_plain(s, case):
    N, K, k, d_in, d_out = (case[q] for q in ("N", "K", "top_k", "d_in", "d_out"))
    R, dtype = N * k, s["x"].dtype
    at, n, cap = _padded(s, K)
    token = torch.div(s["order"][:n].long(), k, rounding_mode="floor")
    w = s["weight"].float()
    xb = torch.zeros(K * cap, d_in, device=w.device)
    xb[at] = s["x"].float()[token]
    xb = xb.view(K, cap, d_in)
    y = torch.zeros(R, d_out, device=w.device)
    y[:n] = torch.bmm(xb, w.transpose(1, 2)).view(K * cap, d_out)[at]
    y = y.to(dtype)
    if case["op"] == "products":
        return [y]
    db = torch.zeros(K * cap, d_out, device=w.device)
    db[at] = s["dy"][:n].float()
    db = db.view(K, cap, d_out)
    d_weight = torch.bmm(db.transpose(1, 2), xb).to(dtype)
    dx_rows = torch.zeros(R + 1, d_in, device=w.device)
    dx_rows[:n] = torch.bmm(db, w).view(K * cap, d_in)[at]
    position = s["position"].long()
    dx = dx_rows[torch.where(position < 0, R, position)].sum(1)
    return [y, dx.to(dtype), d_weight]


def _combine_plain(s, case):
    position = s["position"].long()
    live = position >= 0
    rows = torch.where(live[:, :, None], s["y"].float()[position.clamp(min=0)], 0.0)
    out = (rows * s["weights"][:, :, None]).sum(1).to(s["y"].dtype)
    if case["op"] == "combine":
        return [out]
    g = s["d_out"].float()
    d_weights = (rows * g[:, None, :]).sum(2)
    dy = torch.zeros(s["y"].shape, device=g.device)
    dy[position[live]] = (g[:, None, :] * s["weights"][:, :, None])[live]
    return [out, dy.to(s["y"].dtype), d_weights]


def _group_plain(s, case):
    K, flat = case["K"], s["indices"].reshape(-1).long()
    order = torch.sort(torch.where(flat < 0, K, flat), stable=True)[1]
    offsets = torch.zeros(K + 1, dtype=torch.int64, device=flat.device)
    offsets[1:] = torch.zeros(K + 1, dtype=torch.int64, device=flat.device).scatter_add(
        0, torch.where(flat < 0, K, flat), torch.ones_like(flat))[:K].cumsum(0)
    position = torch.empty_like(flat).scatter(0, order, torch.arange(flat.numel(), device=flat.device))
    position = torch.where(flat < 0, -1, position)
    return [order.int(), offsets.int(), position.int().view(s["indices"].shape)]


# ------------------------------------------------------------------ the framework's calls
def _run_own(s, case):
    from flashgmm_b200 import flash_gmm_native as C
    op = case["op"]
    if op in ("route", "route_train"):
        w, idx = C.route_experts(s["scores"], case["top_k"], score_func=case["score_func"], bias=s["bias"], n_groups=case["n_groups"],
                                 top_groups=case["top_groups"], renormalize=case["renormalize"], scale=case["scale"])
        if op == "route":
            return [w, idx]
        return [w, idx, C.route_experts_backward(s["d_weights"], s["scores"], idx, score_func=case["score_func"],
                                                 renormalize=case["renormalize"], scale=case["scale"])]
    if op == "group":
        return list(C.group_routes(s["indices"], case["K"]))
    routes = C.Routes(s["order"], s["offsets"], s["position"])
    if op in ("products", "products_train"):
        y = C.expert_products(s["x"], s["weight"], routes)
        if op == "products":
            return [y]
        return [y, *C.expert_products_backward(s["dy"], s["x"], s["weight"], routes)]
    out = C.combine_experts(s["y"], s["weights"], routes)
    if op == "combine":
        return [out]
    return [out, *C.combine_experts_backward(s["d_out"], s["y"], s["weights"], routes)]


def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    op = case["op"]
    plain = _route_plain if op.startswith("route") else _group_plain if op == "group" else _products_plain if op.startswith("products") else _combine_plain
    return plain(state, case)


def work(case):
    N, K, k, op = case["N"], case["K"], case["top_k"], case["op"]
    R = N * k
    size = 4 if case.get("dtype", "float32") == "float32" else 2
    if op in ("route", "route_train"):
        scores = N * K * size
        if op == "route":
            return {"bytes": scores + 8 * R + (4 * K if case["bias"] else 0), "flops": 6 * N * K}
        return {"bytes": 2 * scores + 12 * R + (4 * K if case["bias"] else 0), "flops": 8 * N * K}
    if op == "group":
        return {"bytes": 12 * R + 4 * (K + 1), "flops": R}
    d_out = case["d_out"]
    if op in ("products", "products_train"):
        d_in = case["d_in"]
        met = min(K, R)
        x, w, y, flops = N * d_in * size, met * d_in * d_out * size, R * d_out * size, 2 * R * d_in * d_out
        if op == "products":
            return {"bytes": x + w + y + 4 * R + 4 * (K + 1), "flops": flops}
        return {"bytes": 2 * x + w + K * d_in * d_out * size + 2 * y + 8 * R + 4 * (K + 1), "flops": 3 * flops}
    y, out = R * d_out * size, N * d_out * size
    if op == "combine":
        return {"bytes": y + out + 8 * R, "flops": 2 * R * d_out}
    return {"bytes": 2 * y + 2 * out + 12 * R, "flops": 5 * R * d_out}


# ------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definition in 64 bits, point by point or expert by expert."""
    s = prepare(case, seed)
    N, K, k, op = case["N"], case["K"], case["top_k"], case["op"]
    if op in ("route", "route_train"):
        z = s["scores"].double()
        bias = None if s["bias"] is None else s["bias"].double()
        func, per = case["score_func"], K // case["n_groups"]
        live = z > -float("inf")  # false for NaN too
        zm = torch.where(live, z, torch.full_like(z, -float("inf")))
        if func == "softmax":
            value = torch.exp(zm - torch.logsumexp(zm, 1, keepdim=True))
        elif func == "sigmoid":
            value = torch.exp(-torch.logaddexp(torch.zeros_like(z), -zm))
        else:
            value = z
        value = torch.where(live, value, torch.zeros_like(value))
        if bias is None and case["n_groups"] == 1:
            rank = zm.clone()
        else:
            rank = torch.where(live, value if bias is None else value + bias, -float("inf"))
        if case["n_groups"] > 1:
            total = torch.full((N, case["n_groups"]), -float("inf"), dtype=torch.float64, device=z.device)
            for g in range(case["n_groups"]):
                part = rank[:, g * per:(g + 1) * per]
                first, at = part.max(1)
                rest = part.scatter(1, at[:, None], -float("inf")).max(1)[0]
                total[:, g] = first + torch.where(rest == -float("inf"), torch.zeros_like(rest), rest)
            kept = torch.zeros_like(total, dtype=torch.bool)
            for _ in range(case["top_groups"]):
                at = (total == total.amax(1, keepdim=True)).int().argmax(1)
                kept[torch.arange(N, device=z.device), at] = True
                total = torch.where(kept, torch.full_like(total, -float("inf")), total)
            rank = torch.where(kept.repeat_interleave(per, 1), rank, -float("inf"))
        idx = torch.empty(N, k, dtype=torch.int64, device=z.device)
        for j in range(k):
            most = rank.amax(1, keepdim=True)
            at = (rank == most).int().argmax(1)
            idx[:, j] = torch.where(most[:, 0] == -float("inf"), -1, at)
            rank = rank.scatter(1, at[:, None], -float("inf"))
        there = idx >= 0
        at = idx.clamp(min=0)
        w = torch.where(there, value.gather(1, at), 0.0)
        total = w.sum(1, keepdim=True)
        scale = case["scale"]
        share = torch.where(total == 0, 0.0, w / total)
        weights = scale * (share if case["renormalize"] else w)
        if op == "route":
            return [weights, idx.int()]
        g = torch.where(there, s["d_weights"].double() * scale, 0.0)
        # d value of the chosen, then through the score function
        dv = torch.where(total == 0, 0.0, (g - (share * g).sum(1, keepdim=True)) / total) if case["renormalize"] else g
        dvalue = torch.zeros_like(z).scatter_add(1, at, torch.where(there, dv, 0.0))
        if func == "softmax":
            dz = value * (dvalue - (dvalue * value).sum(1, keepdim=True))
        elif func == "sigmoid":
            dz = dvalue * value * (1.0 - value)
        else:
            dz = dvalue
        return [weights, idx.int(), dz]
    if op == "group":
        flat = s["indices"].cpu().numpy().reshape(-1)
        lists = [np.flatnonzero(flat == e) for e in range(K)]
        offsets = np.concatenate([[0], np.cumsum([len(a) for a in lists])]).astype(np.int32)
        order = np.concatenate(lists + [np.flatnonzero(flat < 0)]).astype(np.int32)
        position = np.full(flat.shape, -1, np.int32)
        position[order[:offsets[-1]]] = np.arange(offsets[-1])
        return [order, offsets, position.reshape(N, k)]
    offsets, order = s["offsets"].tolist(), s["order"].long()
    if op in ("products", "products_train"):
        x, R = s["x"].double(), N * k
        y = torch.zeros(R, case["d_out"], dtype=torch.float64, device=x.device)
        dx, dw = torch.zeros_like(x), torch.zeros(s["weight"].shape, dtype=torch.float64, device=x.device)
        for e in range(K):
            a, b = offsets[e], offsets[e + 1]
            if a == b:
                continue
            w, token = s["weight"][e].double(), order[a:b] // k
            y[a:b] = x[token] @ w.T
            if op == "products_train":
                dy = s["dy"][a:b].double()
                dw[e] = dy.T @ x[token]
                dx.index_add_(0, token, dy @ w)
        return [y] if op == "products" else [y, dx, dw]
    n = offsets[-1]
    y, w = s["y"].double(), s["weights"].double().reshape(-1)
    out = torch.zeros(N, case["d_out"], dtype=torch.float64, device=y.device)
    ids = order[:n]
    out.index_add_(0, ids // k, y[:n] * w[ids][:, None])
    if op == "combine":
        return [out]
    g = s["d_out"].double()[ids // k]
    dy, dw = torch.zeros_like(y), torch.zeros_like(w)
    dy[:n] = g * w[ids][:, None]
    dw[ids] = (g * y[:n]).sum(1)
    return [out, dy, dw.view(N, k)]
