"""The expert operators where their values, plans and inputs are at an edge, against their definitions in 64 bits
(tests/experts_ref.py; the roundings that tolerances count are those of tests/test_experts_gpu.py)."""
import math

import pytest
import torch

import experts_ref as ref
from experts_ref import F32_MAX, HALF_STEP
from test_experts_gpu import C, DEV, FUNCS, TYPES, close, gen, plan

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------- routing
@pytest.mark.parametrize("func", FUNCS)
@pytest.mark.parametrize("K,k", [(32, 3), (129, 1), (256, 9), (512, 1), (512, 5), (1000, 32), (4096, 4)])
def test_route_many_infinities_and_largest_scores(func, K, k):
    """+inf counts as the largest finite value: among many of both, the lowest indices are chosen."""
    inf = math.inf
    z = torch.randn(6, K, generator=gen(K))
    z[0, :K // 3] = F32_MAX; z[0, K * 2 // 3] = inf
    z[1, 1::2] = F32_MAX; z[1, 2::4] = inf
    z[2, ::2] = inf
    z[3, :] = F32_MAX; z[3, K - 1] = inf
    z[4, K // 2:] = inf; z[4, K // 2 - 1] = F32_MAX
    z[5, :] = torch.finfo(torch.float32).min; z[5, K - 2] = inf
    for renorm in (True, False):
        got = C().route_experts(z.to(DEV), k, score_func=func, renormalize=renorm)
        assert torch.equal(got[1].cpu(), ref.route(z, k, func, renormalize=renorm)[1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K", [20, 512])
def test_route_shares_of_the_largest_values(K, dtype):
    """Given values whose sum is beyond fp32 still have their shares: a sum and a quotient, 2^-24 and 2^-23 each."""
    inf, k = math.inf, 6
    z = torch.rand(5, K, generator=gen(K)).to(dtype)
    z[0, 3] = z[0, 17] = inf
    z[1, :k] = inf
    z[2] = -inf; z[2, 1] = inf; z[2, 4] = inf; z[2, 6] = -1.0
    z[3] = -inf; z[3, 5] = inf; z[3, 6] = inf; z[3, 9] = torch.finfo(dtype).min
    z[4, 2] = torch.finfo(dtype).max; z[4, 8] = torch.finfo(dtype).max; z[4, 9] = torch.finfo(dtype).max / 2
    w, idx = C().route_experts(z.to(DEV), k, score_func="given")
    want = ref.route(z, k, "given")
    assert torch.equal(idx.cpu(), want[1])
    assert ((w.double().cpu() - want[0]).abs() <= 8 * 2.0 ** -23 * want[0].abs() + 2.0 ** -126).all()
    dz = C().route_experts_backward(torch.randn(5, k, generator=gen(1)).to(DEV), z.to(DEV), idx, score_func="given")
    assert torch.isfinite(dz).all()


@pytest.mark.parametrize("G,T", [(1, 1), (4, 3)])
@pytest.mark.parametrize("K,k", [(32, 7), (128, 10), (256, 21), (512, 30)])
def test_route_near_ties_far_below_the_largest_score(K, k, G, T):
    """exp(z - max) carries the rounding of z - max, |z - max| 2^-24: k - 1 scores 40 or 68 below the row's largest, whose biases
    (1e-4 of the values) bring the values within 2^-15 of each other, are still ordered in 64 bits.  All others are far below."""
    for seed in range(24):
        top, low = ((66.3, -1.7), (40.1, 0.3))[seed % 2]
        g = gen(100 * K + seed)
        at = torch.randperm(K, generator=g)
        z = low - 5 + torch.rand(1, K, generator=g)
        z[0, at[:k - 1]] = low + 1e-4 * torch.rand(k - 1, generator=g)
        z[0, at[-1]] = top
        s = torch.softmax(z.double(), 1)[0]
        bias = torch.zeros(K)
        bias[at[:k - 1]] = (s[at[0]] * (1 + (torch.rand(k - 1, generator=g).double() - 0.5) * 2.0 ** -15) - s[at[:k - 1]]).float()
        got = C().route_experts(z.to(DEV), k, bias=bias.to(DEV), n_groups=G, top_groups=T)
        want = ref.route(z, k, "softmax", bias.double(), G, T)
        assert torch.equal(got[1].cpu(), want[1]), seed


# ------------------------------------------------------------------------------- inputs
@pytest.mark.parametrize("strided", [False, True])
def test_negated_views_are_read_by_value(strided):
    """A view whose memory holds the opposite sign, as the imaginary part of a conjugate is one."""
    def negated(*shape, seed):
        re, im = (torch.randn(*shape, generator=gen(seed + i)).to(DEV) for i in range(2))
        return torch.complex(re, im).conj().imag if strided else torch._neg_view(im)
    N, K, k, d = 40, 6, 2, 16
    z, x, w, dy, wt, b = (negated(*s, seed=10 * i) for i, s in enumerate(((N, K), (N, d), (K, d, d), (N * k, d), (N, k), (K,))))
    assert all(t.is_neg() for t in (z, x, w, dy, wt, b))
    plain = [t.clone().resolve_neg() for t in (z, x, w, dy, wt, b)]
    results = []
    for zi, xi, wi, gi, ti, bi in ((z, x, w, dy, wt, b), plain):
        weights, idx = C().route_experts(zi, k, bias=bi)
        routes = C().group_routes(idx, K)
        results.append([weights, idx, C().route_experts_backward(ti, zi, idx), C().expert_products(xi, wi, routes),
                        *C().expert_products_backward(gi, xi, wi, routes), C().combine_experts(gi, ti, routes),
                        *C().combine_experts_backward(xi, gi, ti, routes)])
    for a, c in zip(*results):
        assert torch.equal(a, c)


def test_derivatives_that_are_not_recorded_are_refused():
    """Forward-mode, batched and traced tensors are refused: nothing drops their derivative in silence or reads through
    pointers that they do not have."""
    import torch.autograd.forward_ad as fw
    from torch._subclasses.fake_tensor import FakeTensorMode
    z, x, w = torch.randn(6, 8, device=DEV), torch.randn(6, 16, device=DEV), torch.randn(8, 4, 16, device=DEV)
    weights, idx = C().route_experts(z, 2)
    routes = C().group_routes(idx, 8)
    y = C().expert_products(x, w, routes)
    calls = [(lambda t: C().route_experts(t, 2)[0], z), (lambda t: C().route_experts(z, 2, bias=t)[0], torch.zeros(8, device=DEV)),
             (lambda t: C().route_experts_backward(t, z, idx), weights), (lambda t: C().expert_products(t, w, routes), x),
             (lambda t: C().expert_products(x, t, routes), w), (lambda t: C().expert_products_backward(t, x, w, routes)[0], y),
             (lambda t: C().combine_experts(t, weights, routes), y), (lambda t: C().combine_experts(y, t, routes), weights),
             (lambda t: C().combine_experts_backward(y[:6].clone(), t, weights, routes)[0], y)]
    for call, t in calls:
        with pytest.raises(RuntimeError):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))
        with pytest.raises(RuntimeError):
            torch.func.vmap(call)(t[None].clone())
        for leaf in (t.clone(), t.clone().requires_grad_()):
            with fw.dual_level(), pytest.raises(RuntimeError):
                call(fw.make_dual(leaf, torch.ones_like(t)))
        call(t)


# -------------------------------------------------------------------------------- plans
def stale(*shape):
    """Leaves NaN in the memory that the next results and workspaces come from."""
    for s in shape:
        torch.full((s,), float("nan"), device=DEV)
    torch.cuda.synchronize()


PATHS = [(torch.float32, 30, 2, 64, 64, 64), (torch.float32, 90, 2, 40, 33, 150), (torch.bfloat16, 30, 2, 64, 63, 64),
         (torch.float32, 300, 2, 4, 128, 72), (torch.bfloat16, 300, 2, 4, 64, 136), (torch.float16, 260, 3, 5, 130, 20)]


@pytest.mark.parametrize("dtype,N,k,K,d_in,d_out", PATHS)
def test_dx_of_a_plan_whose_offsets_end_early(dtype, N, k, K, d_in, d_out):
    """Rows behind offsets[K] belong to no expert, whatever position says of them: they give dx nothing."""
    x, w = torch.randn(N, d_in, generator=gen(1)).to(dtype), torch.randn(K, d_out, d_in, generator=gen(2)).to(dtype)
    dy = torch.randn(N * k, d_out, generator=gen(3)).to(dtype)
    whole = C().group_routes(plan(N, k, K, 3).to(DEV), K)
    for end in (0, 1, N, N * k):
        routes = whole._replace(offsets=whole.offsets.clamp(max=end))
        order, offsets = routes.order.cpu(), routes.offsets.cpu()
        _, _, dx, dxa, dw, dwa = ref.products(x, w, order, offsets, k, dy)
        stale(*[1 << i for i in range(10, 25)])
        gx, gw = C().expert_products_backward(dy.to(DEV), x.to(DEV), w.to(DEV), routes)
        close(gx, dx, dxa, d_out + k, dtype, "dx")
        close(gw, dw, dwa, N * k, dtype, "dw")


@pytest.mark.parametrize("dtype,N,k,K,d_in,d_out", PATHS)
def test_dx_of_a_plan_whose_offsets_do_not_ascend(dtype, N, k, K, d_in, d_out):
    """Such a plan's results are nobody's, but they are made of its inputs: no stale memory is read."""
    x, w = torch.randn(N, d_in, generator=gen(1)).to(dtype), torch.randn(K, d_out, d_in, generator=gen(2)).to(dtype)
    dy = torch.randn(N * k, d_out, generator=gen(3)).to(dtype)
    whole = C().group_routes(torch.randint(0, K, (N, k), generator=gen(4), dtype=torch.int32).to(DEV), K)
    for seed in range(3):
        off = torch.randint(-5, N * k + 5, (K + 1,), generator=gen(seed), dtype=torch.int32)
        off[0], off[K] = 0, N * k
        routes = whole._replace(offsets=off.to(DEV))
        stale(*[1 << i for i in range(10, 25)])
        assert torch.isfinite(C().expert_products(x.to(DEV), w.to(DEV), routes)).all()
        gx, gw = C().expert_products_backward(dy.to(DEV), x.to(DEV), w.to(DEV), routes)
        assert torch.isfinite(gx).all() and torch.isfinite(gw).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_plan_in_which_half_of_the_experts_claim_every_row(dtype):
    """2,048 times the tiles of a plan that ascends, counted up to what 32 bits hold."""
    N, k, K, d = 9000, 2, 4096, 64
    x, w = torch.randn(N, d, generator=gen(1)).to(dtype).to(DEV), torch.randn(1, d, d, generator=gen(2)).to(dtype).to(DEV).expand(K, d, d).contiguous()
    dy = torch.randn(N * k, d, generator=gen(3)).to(dtype).to(DEV)
    whole = C().group_routes(torch.zeros(N, k, dtype=torch.int32, device=DEV), K)
    off = torch.zeros(K + 1, dtype=torch.int32)
    off[1::2] = N * k
    off[K] = N * k
    routes = whole._replace(offsets=off.to(DEV))
    stale(*[1 << i for i in range(10, 25)])
    # every expert holds the same matrix: whichever of them writes a row last, it is the same row
    assert torch.equal(C().expert_products(x, w, routes), C().expert_products(x, w, whole))
    gx, gw = C().expert_products_backward(dy, x, w, routes)
    assert torch.equal(gx, C().expert_products_backward(dy, x, w, whole)[0])
    assert gw.shape == w.shape
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,k,d", [(5, 3, 7), (40, 2, 64), (300, 4, 264)])
def test_weights_gradient_of_slots_that_order_leaves_out(dtype, N, k, d):
    """A plan of a part of the experts: the other routes' places in order hold no route, and their slots' gradient is 0."""
    K = 8
    idx = torch.randint(0, K, (N, k), generator=gen(N), dtype=torch.int32)
    routes = C().group_routes(idx.to(DEV), K)
    y, wt, g = torch.randn(N * k, d, generator=gen(1)).to(dtype), torch.randn(N, k, generator=gen(2)), torch.randn(N, d, generator=gen(3)).to(dtype)
    away = idx >= 5
    order = torch.where(away.flatten()[routes.order.long().cpu()], -1, routes.order.cpu())
    position = torch.where(away, -1, routes.position.cpu())
    part = routes._replace(order=order.to(DEV), position=position.to(DEV))
    _, _, dy, dw, dwa = ref.combine(y, wt, position, g)
    gd, yd, wd = g.to(DEV), y.to(DEV), wt.to(DEV)

    def without_position():
        from flashgmm_b200 import _lib
        gy, gw = torch.full_like(yd, math.nan), torch.full_like(wd, math.nan)
        at = [t.data_ptr() for t in (gd, yd, wd, part.order, part.offsets, gy, gw)]
        _lib.check(_lib.load().fgmm_combine_experts_backward(at[0], at[1], TYPES.index(dtype), N, d, *at[2:5], K, k, at[5], at[6],
                                                             torch.cuda.current_stream().cuda_stream))
        return gy, gw

    for call in (lambda: C().combine_experts_backward(gd, yd, wd, part), without_position) * 2:
        stale(*[1 << i for i in range(2, 16)])
        gy, gw = call()
        assert (gw.cpu()[away] == 0).all() and (gy.cpu()[order < 0] == 0).all()
        assert ((gw.double().cpu() - dw).abs() <= (d / 32 + 8) * 2.0 ** -24 * 2 * dwa).all()
        assert ((gy.double().cpu() - dy).abs() <= (2.0 ** -24 + HALF_STEP[dtype]) * dy.abs() * 1.001 + 2.0 ** -24 * (dtype == torch.float16)).all()


# ------------------------------------------------------------------------------ products
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,k,K,d_in,d_out", [(300, 2, 4, 64, 16), (40, 2, 32, 64, 16), (30, 2, 64, 63, 9), (2100, 3, 3, 128, 8), (700, 4, 16, 100, 40)])
def test_dx_rounds_once(N, k, K, d_in, d_out, dtype):
    """A point's rows cancel almost: one rounding of their sum is far below a rounding of each row."""
    g = gen(N + K)
    w = torch.randn(1, d_out, d_in, generator=g).expand(K, -1, -1) + torch.randn(K, d_out, d_in, generator=g) * 2.0 ** -6
    w, x = w.to(dtype), torch.randn(N, d_in, generator=g).to(dtype)
    idx = plan(N, k, K, N + K, dropped=False)
    routes = C().group_routes(idx.to(DEV), K)
    order = routes.order.cpu().long()
    sign = torch.tensor([1.0, -1.0])[order % k % 2]
    dy = (torch.randn(N, d_out, generator=g)[order // k] * sign[:, None] * 16).to(dtype)
    _, _, dx, dxa, _, _ = ref.products(x, w, routes.order.cpu(), routes.offsets.cpu(), k, dy)
    gx = C().expert_products_backward(dy.to(DEV), x.to(DEV), w.to(DEV), routes, need_dweight=False)[0]
    close(gx, dx, dxa, d_out + k, dtype, "dx")


@pytest.mark.parametrize("dtype,N,k,K,d_in,d_out", [(torch.float32, 300, 1, 64, 40, 72), (torch.float32, 190, 2, 64, 1030, 33), (torch.bfloat16, 250, 1, 64, 63, 40)])
def test_few_rows_of_one_popular_expert(dtype, N, k, K, d_in, d_out):
    """Few rows an expert on average, and one of them has most."""
    idx = torch.full((N, k), 7, dtype=torch.int32)
    idx[::5, 0] = torch.randint(0, K, (len(idx[::5]),), generator=gen(1), dtype=torch.int32)
    idx[:, 1:] = (idx[:, :1] + 1) % K
    x, w = torch.randn(N, d_in, generator=gen(2)).to(dtype), (torch.randn(K, d_out, d_in, generator=gen(3)) / d_in ** 0.5).to(dtype)
    dy = torch.randn(N * k, d_out, generator=gen(4)).to(dtype)
    routes = C().group_routes(idx.to(DEV), K)
    y, ya, dx, dxa, dw, dwa = ref.products(x, w, routes.order.cpu(), routes.offsets.cpu(), k, dy)
    close(C().expert_products(x.to(DEV), w.to(DEV), routes), y, ya, d_in, dtype, "y")
    gx, gw = C().expert_products_backward(dy.to(DEV), x.to(DEV), w.to(DEV), routes)
    close(gx, dx, dxa, d_out + k, dtype, "dx")
    close(gw, dw, dwa, N * k, dtype, "dw")


HALVES = [torch.float16, torch.bfloat16]


def one_sign(*shape, seed, dtype):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.rand(*shape, generator=g, device=DEV) * 0.125 + 0.0625).to(dtype)


def check_one_sign(got, want, dtype, segments):
    """Tensor memory truncates, by less than 2^-23 of the running sum for 8 elements of the contraction: of 8,192 elements of
    one sign less than 1,024 2^-23 / 2 of their sum.  The segments' sums are added in fp32, and the result rounds once."""
    off = ((got.double() - want) / want).abs()
    lim = HALF_STEP[dtype] + 2.0 ** -14 + segments * 2.0 ** -24
    assert float(off.max()) <= lim * 1.001, (float(off.max()), lim)


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("K,d_in,d_out,R", [(64, 256, 896, 1 << 20), (4, 128, 128, 1 << 20), (4, 100, 130, 300001), (64, 512, 1024, 8193), (64, 512, 1024, 70000),
                                               (4, 2560, 1280, 65613)])
def test_weights_gradient_of_very_many_rows_of_one_sign(K, d_in, d_out, R, dtype):
    x, dy = one_sign(R, d_in, seed=1, dtype=dtype), one_sign(R, d_out, seed=2, dtype=dtype)
    idx = torch.full((R, 1), 2, dtype=torch.int32, device=DEV)
    idx[::64] = 3
    routes = C().group_routes(idx, K)
    gw = C().expert_products_backward(dy, x, torch.zeros(K, d_out, d_in, device=DEV, dtype=dtype), routes, need_dx=False)[1]
    for e in (2, 3):
        of = slice(int(routes.offsets[e]), int(routes.offsets[e + 1]))
        want = sum(a.double().T @ b.double() for a, b in zip(dy[of].chunk(16), x[routes.order[of].long()].chunk(16)))
        check_one_sign(gw[e], want, dtype, R // 8192 + 1)
    assert (gw[:2] == 0).all() and (gw[4:] == 0).all()


@pytest.mark.parametrize("dtype", HALVES)
@pytest.mark.parametrize("d,other", [(8200, 136), (20003, 33), (65536, 520), (1 << 18, 128)])
def test_products_of_very_wide_rows_of_one_sign(d, other, dtype):
    N, K = 333, 2
    idx = torch.arange(N, dtype=torch.int32, device=DEV)[:, None] % K
    routes = C().group_routes(idx, K)
    rows = routes.order.long()
    at = [slice(int(a), int(b)) for a, b in zip(routes.offsets[:-1], routes.offsets[1:])]
    x, w = one_sign(N, d, seed=1, dtype=dtype), one_sign(K, other, d, seed=2, dtype=dtype) / 16
    y = C().expert_products(x, w, routes)
    for e in range(K):
        check_one_sign(y[at[e]], x[rows[at[e]]].double() @ w[e].double().T, dtype, d // 8192 + 1)
    dy, w = one_sign(N, d, seed=3, dtype=dtype), one_sign(K, d, other, seed=4, dtype=dtype) / 16
    dx = C().expert_products_backward(dy, torch.zeros(N, other, device=DEV, dtype=dtype), w, routes, need_dweight=False)[0]
    for e in range(K):
        check_one_sign(dx[rows[at[e]]], dy[at[e]].double() @ w[e].double(), dtype, d // 8192 + 1)


@pytest.mark.parametrize("dtype", HALVES)
def test_infinities_in_wide_rows_stay_where_they_belong(dtype):
    N, K, d, d_out = 300, 3, 20000, 72
    x, w = torch.randn(N, d, generator=gen(1)), torch.randn(K, d_out, d, generator=gen(2)) / 128
    x[5, 3], x[6, 9000], x[7, 3], x[7, 19999], x[8, 12000] = math.inf, -math.inf, math.inf, math.inf, math.nan
    x, w = x.to(dtype).to(DEV), w.to(dtype).to(DEV)
    routes = C().group_routes(torch.arange(N, dtype=torch.int32, device=DEV)[:, None] % K, K)
    y = C().expert_products(x, w, routes)
    place = routes.position[:, 0].long()
    want = torch.stack([(x[n].double() * w[n % K].double()).sum(1) for n in range(5, 9)])
    got = y[place[5:9]].double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.isinf(), want.isinf())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    rest = [n for n in range(N) if not 5 <= n < 9]
    assert torch.isfinite(y[place[rest]]).all()


# --------------------------------------------------------------- waits that have run out
def a_wait_ran_out():
    """What the products' kernels leave behind: a code in the device's word of host memory."""
    from flashgmm_b200 import _lib
    word = _lib.load().fgmm_expert_error_word()
    word[0] = 3
    return word


def test_a_wait_that_ran_out_is_raised_by_the_next_product():
    from flashgmm_b200 import _lib
    idx = torch.randint(0, 4, (200, 2), generator=gen(1), dtype=torch.int32).to(DEV)
    routes = C().group_routes(idx, 4)
    x, w = torch.randn(200, 64, device=DEV).bfloat16(), torch.randn(4, 72, 64, device=DEV).bfloat16()
    want = C().expert_products(x, w, routes)
    dx, dw = C().expert_products_backward(want, x, w, routes)
    leaf = x.clone().requires_grad_()
    calls = [lambda: C().expert_products(x, w, routes), lambda: C().expert_products_backward(want, x, w, routes),
             lambda: C().expert_products(leaf, w, routes), lambda: C().expert_products(x[:1, :8].float(), w[:, :8, :8].float(),
                                                                                       C().group_routes(idx[:1], 4))]
    for call in calls:
        word = a_wait_ran_out()
        with pytest.raises(RuntimeError, match="bounded wait"):
            call()
        assert word[0] == 0
        call()
    y = C().expert_products(leaf, w, routes)
    a_wait_ran_out()
    with pytest.raises(RuntimeError, match="bounded wait"):
        y.backward(want)
    a_wait_ran_out()
    with pytest.raises(_lib.DeviceWaitError):
        C().check_expert_products()
    C().check_expert_products()
    assert torch.equal(C().expert_products(x, w, routes), want)
    assert all(torch.equal(a, b) for a, b in zip(C().expert_products_backward(want, x, w, routes), (dx, dw)))


def test_a_wait_that_ran_out_and_a_capture():
    """A capture does not clear the word: the call fails, and the next call outside of it fails too, once."""
    idx = torch.randint(0, 4, (200, 2), generator=gen(1), dtype=torch.int32).to(DEV)
    x, w = torch.randn(200, 64, device=DEV), torch.randn(4, 72, 64, device=DEV)
    routes = C().group_routes(idx, 4)
    want = C().expert_products(x, w, routes)
    torch.cuda.synchronize()
    word = a_wait_ran_out()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="bounded wait"):
        with torch.cuda.graph(graph):
            x + 1
            C().expert_products(x, w, routes)
    assert word[0] == 3
    with pytest.raises(RuntimeError, match="bounded wait"):
        C().expert_products(x, w, routes)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = C().expert_products(x, w, routes)
    graph.replay()
    assert torch.equal(y, want)


def test_a_fit_does_not_answer_for_the_products():
    from flashgmm_b200 import native_wrapper
    from flashgmm_b200.data import make_mixture
    N, K, d = 2000, 16, 32
    X = make_mixture(N, K, d, seed=3)[0].to(DEV)
    m = native_wrapper.NativeFlashGMM(K, d, max_iter=3)
    weight = torch.randn(K, 8, d, device=DEV)
    word = a_wait_ran_out()
    m.fit(X)
    assert word[0] == 3
    with pytest.raises(RuntimeError, match="bounded wait"):
        m.mix_experts(X, weight, 2)
    assert torch.isfinite(m.mix_experts(X, weight, 2)).all()
