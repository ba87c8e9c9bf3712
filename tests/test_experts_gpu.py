"""The expert operators on the GPU against their definitions in 64 bits (tests/experts_ref.py).

Tolerances count roundings.  HALF_STEP[t] is a type's largest relative rounding.  Sums of d products in fp32:
each of d additions and products rounds once, and tensor-core accumulation may truncate (a whole step),
so |error| <= 2 d 2^-23 sum |a b| (half of that on the CUDA cores), and half a step of the output type.
The bulk is held to a norm: the roundings of different products are independent or drain in fp32
segments, which keeps the 2-norm of the error below 2^-19 of the sums of magnitudes' norm.
"""
import math

import pytest
import torch

import experts_ref as ref
from experts_ref import HALF_STEP

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.bfloat16, torch.float16]
FUNCS = ["softmax", "sigmoid", "given"]


def C():
    from flashgmm_b200 import flash_gmm_native
    return flash_gmm_native


def gen(seed):
    return torch.Generator().manual_seed(seed)


def scores_of(N, K, dtype, seed, func="softmax"):
    z = torch.randn(N, K, generator=gen(seed)) * 1.5
    if func == "given":
        z = torch.softmax(4 * z, 1)
    return z.to(dtype)


def check_route(z, got, want, func, scale):
    """Equal indices; weights within the roundings of exp and its argument (|z - max| 2^-24 each), the
    sum over K and the division: (2 spread + 16 + log2 K) 2^-23 relative, K's sum being pairwise over the lanes."""
    w, idx = got[0].double().cpu(), got[1].cpu()
    assert w.shape == want[0].shape and idx.dtype == torch.int32
    bad = (idx != want[1]).any(1).nonzero().flatten()
    assert bad.numel() == 0, (bad[:5], idx[bad[:2]], want[1][bad[:2]])
    zf = z.float().cpu()
    fin = zf[torch.isfinite(zf) & (zf.abs() < 1e30)]
    spread = float(fin.max() - fin.min()) if fin.numel() and func != "given" else 0.0
    K = z.shape[1]
    rtol = (2 * spread + 16 + K / 32 + math.log2(32)) * 2.0 ** -23
    assert ((w - want[0]).abs() <= rtol * want[0].abs() + 1e-37 * scale).all(), float(
        ((w - want[0]).abs() / want[0].abs().clamp(min=1e-37)).max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K,k", [(1, 1, 1), (1, 256, 8), (37, 7, 3), (130, 33, 8), (65, 100, 1), (9, 1024, 16), (5, 1025, 4),
                                   (3, 4096, 32), (64, 64, 31)])
def test_route_leading_experts(N, K, k, dtype):
    for func in FUNCS:
        for renorm, scale in ((True, 1.0), (False, 2.5)):
            z = scores_of(N, K, dtype, N + K + k, func)
            got = C().route_experts(z.to(DEV), k, score_func=func, renormalize=renorm, scale=scale)
            want = ref.route(z, k, func, renormalize=renorm, scale=scale)
            check_route(z, got, want, func, scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K,k,G,T", [(50, 256, 8, 8, 4), (33, 64, 6, 4, 1), (21, 96, 4, 3, 2), (40, 30, 5, 10, 3), (12, 32, 4, 32, 5),
                                       (7, 1000, 8, 8, 3), (5, 2048, 8, 16, 4), (6, 64, 32, 2, 1), (6, 20, 20, 4, 2)])
def test_route_groups_and_bias(N, K, k, G, T, dtype):
    for func in FUNCS:
        for with_bias in (False, True):
            z = scores_of(N, K, dtype, 3 * N + K, func)
            bias = torch.randn(K, generator=gen(5)) * 0.05 if with_bias else None
            got = C().route_experts(z.to(DEV), k, score_func=func, bias=None if bias is None else bias.to(DEV), n_groups=G,
                                    top_groups=T, renormalize=True, scale=2.5)
            want = ref.route(z, k, func, None if bias is None else bias.double(), G, T, True, 2.5)
            check_route(z, got, want, func, 2.5)


@pytest.mark.parametrize("func", FUNCS)
@pytest.mark.parametrize("G,T", [(1, 1), (4, 2)])
def test_route_ties_and_near_ties(func, G, T):
    """Equal values go to the lowest index; values closer than fp32 resolves are ordered in 64 bits."""
    N, K, k = 64, 64, 6
    z = torch.randint(-2, 3, (N, K), generator=gen(1)).float() * 0.5
    if func == "given":
        z = z.abs()
    zero_bias, bias = torch.zeros(K), torch.randint(-1, 2, (K,), generator=gen(2)).float() * 2.0 ** -26
    for b in (None, zero_bias, bias):
        got = C().route_experts(z.to(DEV), k, score_func=func, bias=None if b is None else b.to(DEV), n_groups=G, top_groups=T)
        check_route(z, got, ref.route(z, k, func, None if b is None else b.double(), G, T), func, 1.0)
    same = torch.zeros(3, K)
    got = C().route_experts(same.to(DEV), k, score_func=func, bias=zero_bias.to(DEV), n_groups=G, top_groups=T)
    assert got[1].cpu().tolist() == [list(range(k))] * 3


@pytest.mark.parametrize("func", ["softmax", "sigmoid"])
@pytest.mark.parametrize("N,K,k,G,T", [(40, 64, 6, 4, 2), (33, 30, 5, 1, 1), (21, 100, 2, 1, 1), (20, 256, 3, 1, 1), (40, 256, 8, 8, 4), (20, 256, 1, 8, 4),
                                       (20, 200, 32, 1, 1), (9, 1024, 8, 32, 3), (5, 2048, 8, 16, 3), (20, 20, 20, 4, 2)])
def test_route_equal_and_nearly_equal_together(func, N, K, k, G, T):
    """Rows of few distinct scores: saturated ones, which fp32 values do not tell apart, and neighbours in fp32, many of each."""
    g = gen(N + K + k)
    saturated = 20.0 + torch.randint(0, 5, (N, K), generator=g) * 0.125
    near = 1.0 + torch.randint(0, 4, (N, K), generator=g) * 2.0 ** -23
    small = torch.randint(-1, 2, (K,), generator=g).float() * 2.0 ** -26
    for z in (saturated, near):
        for bias in (None, torch.zeros(K), small):
            got = C().route_experts(z.to(DEV), k, score_func=func, bias=None if bias is None else bias.to(DEV), n_groups=G, top_groups=T)
            check_route(z, got, ref.route(z, k, func, bias, G, T), func, 1.0)


@pytest.mark.parametrize("func", FUNCS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("G,T,with_bias", [(1, 1, False), (1, 1, True), (4, 2, True)])
def test_route_masks(func, dtype, G, T, with_bias):
    """Rows with nothing left, with fewer experts than slots, NaN and infinities in masked and live places,
    a type's lowest value as a mask, and whole groups masked."""
    N, K, k = 24, 32, 5
    inf, low = float("inf"), torch.finfo(dtype).min
    z = scores_of(N, K, dtype, 9, func)
    z[0] = -inf
    z[1] = float("nan")
    z[2, :] = -inf; z[2, 17] = 0.5
    z[3, ::2] = float("nan")
    z[4, 3:] = low
    z[5, :] = low
    z[6, :8] = -inf
    z[7, 8:] = -inf
    z[8, 5] = inf
    z[9, 5] = inf; z[9, 20] = inf
    z[10, :30] = -inf
    bias = torch.randn(K, generator=gen(5)) * 0.05 if with_bias else None
    if with_bias:
        bias[4] = -inf
    for renorm in (True, False):
        got = C().route_experts(z.to(DEV), k, score_func=func, bias=None if bias is None else bias.to(DEV), n_groups=G,
                                top_groups=T, renormalize=renorm)
        want = ref.route(z, k, func, None if bias is None else bias.double(), G, T, renorm)
        if func == "given":  # its weights are the scores: the rows with the lowest or largest value hold no shares
            rows = [n for n in range(N) if n not in (4, 5, 8, 9)]
        elif func == "sigmoid" and renorm:  # shares of values that all underflow are taken as limits: 1 / k each
            rows = [n for n in range(N) if n != 5]
            w5 = got[0][5].cpu()
            assert torch.allclose(w5[got[1][5].cpu() >= 0], torch.full((int((got[1][5] >= 0).sum()),), 1.0 / k), atol=1e-6)
        else:
            rows = list(range(N))
        assert torch.equal(got[1].cpu(), want[1])
        check_route(z[rows], (got[0][rows], got[1][rows]), (want[0][rows], want[1][rows]), func, 1.0)
        assert torch.isfinite(got[0].cpu()[rows]).all()
        assert (got[0].cpu()[got[1].cpu() < 0] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_route_reads_through_strides(dtype):
    wide = scores_of(40, 200, dtype, 4).to(DEV)
    for z in (wide[:, 3:103], wide[::2, :64], wide.t()[:50], wide[:1].expand(9, 200), wide[:, 8:9]):
        k = min(4, z.shape[1])
        a, b = C().route_experts(z, k), C().route_experts(z.contiguous(), k)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        dw = torch.randn(z.shape[0], k, device=DEV)
        assert torch.equal(C().route_experts_backward(dw, z, a[1]), C().route_experts_backward(dw, z.contiguous(), a[1]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,K,k", [(1, 1, 1), (40, 7, 3), (33, 128, 2), (20, 1000, 8), (3, 2500, 4), (2, 4096, 32)])
def test_route_gradient(N, K, k, dtype):
    """Against autograd of the formula in 64 bits.  The chosen scores' part is p (g - sum p g): each factor
    carries the weights' roundings, so |error| <= 2 (spread + 16 + K / 32) 2^-23 scale max |dw|, of sums
    that are at most 2, and half a step of the type."""
    for func in FUNCS:
        for renorm, scale in ((True, 2.5), (False, 1.0)):
            z = scores_of(N, K, dtype, N + K, func)
            dw = torch.randn(N, k, generator=gen(8))
            idx = C().route_experts(z.to(DEV), k, score_func=func, renormalize=renorm, scale=scale)[1]
            got = C().route_experts_backward(dw.to(DEV), z.to(DEV), idx, score_func=func, renormalize=renorm, scale=scale)
            z64 = z.double().requires_grad_()
            ref.weights_of(z64, idx.cpu(), func, renorm, scale).backward(dw.double())
            want = z64.grad
            assert got.dtype == dtype and got.shape == z.shape
            spread = float(z.float().max() - z.float().min()) if func != "given" else 0.0
            size = want.abs().max() if func == "given" else 2 * scale * dw.abs().max()
            tol = 2 * (spread + 16 + K / 32) * 2.0 ** -23 * size + HALF_STEP[dtype] * want.abs() * 1.001 + 2.0 ** -25 * (dtype == torch.float16)
            assert ((got.double().cpu() - want).abs() <= tol).all(), (func, renorm, float((got.double().cpu() - want).abs().max()))


@pytest.mark.parametrize("func", FUNCS)
@pytest.mark.parametrize("renorm", [True, False])
def test_route_gradient_against_differences(func, renorm):
    """d weights along a direction v by central differences of the kernel's own weights: their truncation
    is below eps^2 times the third derivative (< 1 here, |v| <= 1), their roundings below 2^-21 / eps."""
    N, K, k, eps = 16, 24, 4, 2.0 ** -7
    z = scores_of(N, K, torch.float32, 3, func).to(DEV) * (1.0 if func != "given" else 16.0)
    z = torch.sort(z, 1)[0] + torch.arange(K, device=DEV) * 0.25  # the choice does not change within eps
    v = torch.rand(N, K, generator=gen(4)).to(DEV) * 2 - 1
    dw = torch.randn(N, k, generator=gen(5)).to(DEV)
    args = dict(score_func=func, renormalize=renorm)
    up, down = C().route_experts(z + eps * v, k, **args), C().route_experts(z - eps * v, k, **args)
    mid = C().route_experts(z, k, **args)
    assert torch.equal(up[1], mid[1]) and torch.equal(down[1], mid[1])
    num = ((up[0] - down[0]).double() / (2 * eps) * dw).sum(1)
    ana = (C().route_experts_backward(dw, z, mid[1], **args).double() * v).sum(1)
    tol = (eps ** 2 + 2.0 ** -21 / eps * float(mid[0].abs().max().clamp(min=1))) * float(dw.abs().sum(1).max()) * 4
    assert ((num - ana).abs() <= tol).all()


def test_route_gradient_of_masked_and_repeated_slots():
    z = torch.randn(6, 8, generator=gen(1))
    z[0] = -math.inf
    z[1, 2:] = -math.inf
    z[2, 3] = math.nan
    zd = z.to(DEV)
    w, idx = C().route_experts(zd, 3)
    dz = C().route_experts_backward(torch.ones(6, 3, device=DEV) * torch.tensor([1., 2., 3.], device=DEV), zd, idx)
    assert torch.isfinite(dz).all() and (dz[0] == 0).all() and (dz[1, 2:] == 0).all() and dz[2, 3] == 0
    # the same expert in two slots, and slots that no expert fills: the slots' gradients add up
    idx = torch.tensor([[4, 4, -1]] * 6, dtype=torch.int32, device=DEV)
    g = torch.randn(6, 3, device=DEV)
    z2 = torch.randn(6, 8, device=DEV)
    for func in FUNCS:
        got = C().route_experts_backward(g, z2, idx, score_func=func, renormalize=False)
        zz = z2.double().cpu().requires_grad_()
        ref.weights_of(zz, idx.cpu(), func, False, 1.0).backward(g.double().cpu())
        assert torch.allclose(got.double().cpu(), zz.grad, atol=1e-6)
    out_of_range = torch.tensor([[99, -7, 1 << 30]] * 6, dtype=torch.int32, device=DEV)
    assert (C().route_experts_backward(g, z2, out_of_range) == 0).all()


# ------------------------------------------------------------------------------ grouping
@pytest.mark.parametrize("N,k,K", [(1, 1, 1), (37, 4, 64), (2047, 1, 5), (2049, 3, 300), (5000, 8, 1024), (700, 2, 4096), (40000, 2, 17), (4096, 1, 3), (4097, 1, 3),
                                   (350001, 3, 64)])
def test_group_routes(N, k, K):
    idx = torch.randint(-1, K + 1, (N, k), generator=gen(N + K), dtype=torch.int32)  # some without an expert, some outside
    routes = C().group_routes(idx.to(DEV), K)
    for a, b in zip(routes, ref.group(idx, K)):
        assert a.dtype == torch.int32 and torch.equal(a.cpu(), b)


def test_group_routes_of_one_expert_and_of_none():
    for fill in (0, 3, -1, -(1 << 31), (1 << 31) - 1):
        idx = torch.full((3000, 2), fill, dtype=torch.int32)
        for a, b in zip(C().group_routes(idx.to(DEV), 4), ref.group(idx, 4)):
            assert torch.equal(a.cpu(), b)
    idx = torch.randint(0, 9, (50, 6), generator=gen(1), dtype=torch.int32).to(DEV)
    for t in (idx[:, ::2], idx.t(), idx[::3]):  # copied where they are not contiguous
        for a, b in zip(C().group_routes(t, 9), C().group_routes(t.contiguous(), 9)):
            assert torch.equal(a, b)


# ------------------------------------------------------------------------------ products
def plan(N, k, K, seed, dropped=True, spread=0.7):
    """Routes with unevenly wanted experts, some experts without a point, some points without an expert."""
    g = gen(seed)
    wanted = torch.randn(N, K, generator=g) + torch.randn(K, generator=g) * spread
    if K > 3:
        wanted[:, K // 2] = -100.0
    idx = torch.topk(wanted, k, 1)[1].int()
    if dropped and N > 2:
        idx[N // 2] = -1
        idx[N - 1, 0] = -1
    return idx


def close(got, want, size, d, dtype, what):
    """Elementwise bound, and the norm's (see the module's docstring)."""
    err = (got.double().cpu() - want).abs()
    tol = 2 * d * 2.0 ** -23 * size + HALF_STEP[dtype] * want.abs() * 1.001 + (2.0 ** -24 if dtype == torch.float16 else 0)
    assert (err <= tol).all(), (what, float((err - tol).max()), float(err.max()))
    norm = float(err.norm())
    lim = HALF_STEP[dtype] * float(want.norm()) + 2.0 ** -19 * float(size.norm()) + (2.0 ** -24 * want.numel() ** 0.5 if dtype == torch.float16 else 0)
    assert norm <= lim, (what, norm, lim)


SIZES = [(1, 1, 1, 1, 1), (1, 2, 8, 64, 128), (5, 2, 4, 3, 7), (33, 2, 5, 64, 64), (100, 3, 6, 72, 136), (257, 2, 3, 100, 65),
         (300, 4, 16, 128, 128), (64, 1, 64, 256, 320), (700, 2, 4, 520, 264), (1100, 2, 2, 192, 384), (16, 4, 64, 1024, 512),
         (129, 1, 1, 1000, 1016), (40, 2, 3, 1025, 33)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,k,K,d_in,d_out", SIZES)
def test_products_and_gradients(N, k, K, d_in, d_out, dtype):
    g = gen(N + d_in)
    x, w = torch.randn(N, d_in, generator=g).to(dtype), (torch.randn(K, d_out, d_in, generator=g) / d_in ** 0.5).to(dtype)
    dy = torch.randn(N * k, d_out, generator=g).to(dtype)
    routes = C().group_routes(plan(N, k, K, N + K).to(DEV), K)
    order, offsets = routes.order.cpu(), routes.offsets.cpu()
    n_live = int(offsets[-1])
    y, ya, dx, dxa, dw, dwa = ref.products(x, w, order, offsets, k, dy)
    got = C().expert_products(x.to(DEV), w.to(DEV), routes)
    assert got.shape == (N * k, d_out) and got.dtype == dtype
    close(got, y, ya, d_in, dtype, "y")
    assert (got[n_live:] == 0).all()
    # rows of no expert may hold anything
    dyd = dy.to(DEV)
    dyd[n_live:] = float("nan")
    gx, gw = C().expert_products_backward(dyd, x.to(DEV), w.to(DEV), routes)
    # each of a point's rows is rounded to the type before their sum: k more half steps of the rows' sizes
    err = (gx.double().cpu() - dx).abs()
    assert (err <= 2 * d_out * 2.0 ** -23 * dxa + 1.01 * HALF_STEP[dtype] * (dx.abs() + dxa) + 2.0 ** -23).all(), "dx"
    assert float(err.norm()) <= 2.0 ** -19 * float(dxa.norm()) + 3 * HALF_STEP[dtype] * float(dx.norm()) + 2.0 ** -23
    counts = offsets[1:] - offsets[:-1]
    close(gw, dw, dwa, max(1, int(counts.max())), dtype, "dw")
    assert (gw[(counts == 0).to(DEV)] == 0).all()
    assert C().expert_products_backward(dyd, x.to(DEV), w.to(DEV), routes, need_dx=False)[0] is None
    only = C().expert_products_backward(dyd, x.to(DEV), w.to(DEV), routes, need_dweight=False)
    assert only[1] is None and torch.equal(only[0], gx)


@pytest.mark.parametrize("dtype", TYPES)
def test_products_keep_infinities_where_they_belong(dtype):
    """An infinite or NaN row reaches its own results only, although tiles hold several experts' rows."""
    N, k, K, d_in, d_out = 90, 2, 5, 72, 80
    x, w = torch.randn(N, d_in, generator=gen(1)).to(dtype), torch.randn(K, d_out, d_in, generator=gen(2)).to(dtype)
    dy = torch.randn(N * k, d_out, generator=gen(3)).to(dtype)
    routes = C().group_routes(plan(N, k, K, 4).to(DEV), K)
    order, offsets = routes.order.cpu(), routes.offsets.cpu()
    base = C().expert_products(x.to(DEV), w.to(DEV), routes)
    x2 = x.clone()
    x2[7] = float("nan")
    x2[8, 3] = float("inf")
    got = C().expert_products(x2.to(DEV), w.to(DEV), routes)
    own = torch.isin(order // k, torch.tensor([7, 8])).to(DEV)
    assert torch.equal(got[~own], base[~own]) and not torch.isfinite(got[own][: 1]).any()
    # one expert's dy is not finite: the other experts' gradients are as before
    e = int((offsets[1:] - offsets[:-1]).argmax())
    a, b = int(offsets[e]), int(offsets[e + 1])
    gx0, gw0 = C().expert_products_backward(dy.to(DEV), x.to(DEV), w.to(DEV), routes)
    dy2 = dy.clone()
    dy2[a:b] = float("inf")
    gx, gw = C().expert_products_backward(dy2.to(DEV), x.to(DEV), w.to(DEV), routes)
    others = [i for i in range(K) if i != e]
    assert torch.equal(gw[others], gw0[others])
    untouched = torch.ones(N, dtype=torch.bool)
    untouched[(order[a:b] // k).long()] = False
    assert torch.equal(gx[untouched.to(DEV)], gx0[untouched.to(DEV)])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,k,K,d_in,d_out", [(21, 3, 32, 136, 256), (9, 5, 40, 72, 200), (12, 32, 40, 64, 72), (50, 2, 4096, 64, 64), (7, 3, 4096, 20, 31),
                                              (2100, 3, 3, 128, 128), (515, 7, 9, 320, 256), (65, 1, 1, 1025, 2050)])
def test_products_of_more_plans(N, k, K, d_in, d_out, dtype):
    """Many slots, odd numbers of them, the largest number of experts, one expert with everything."""
    test_products_and_gradients(N, k, K, d_in, d_out, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N", [3, 300])
def test_products_of_infinite_and_largest_values(N, dtype):
    """Infinite, NaN and largest entries in either operand give what 64 bits give, on the CUDA cores (few rows an expert) and on
    the tensor cores.  (The scaled columns keep the largest value's products within the type.)"""
    k, K, d_in, d_out = 1, 4, 136, 72
    x, w = torch.randn(N, d_in, generator=gen(1)), torch.randn(K, d_out, d_in, generator=gen(2))
    dy = torch.randn(N * k, d_out, generator=gen(3))
    w[:, :, 5] *= 2.0 ** (-100 if dtype != torch.float16 else -14)
    x, w, dy = x.to(dtype), w.to(dtype), dy.to(dtype)
    x[0, 3], x[1, 130], x[2, 7] = float("inf"), float("-inf"), float("nan")
    if N > 3:
        x[3:100:2, 5], x[4:100:2, 5] = torch.finfo(dtype).max, torch.finfo(dtype).min
        w[1, 2, 9] = float("-inf")
    idx = torch.arange(N * k, dtype=torch.int32).reshape(N, k) % K
    routes = C().group_routes(idx.to(DEV), K)
    order, offsets = routes.order.cpu(), routes.offsets.cpu()
    y, ya, dx, dxa, dw, dwa = ref.products(x, w, order, offsets, k, dy)
    gx, gw = C().expert_products_backward(dy.to(DEV), x.to(DEV), w.to(DEV), routes)
    counts = offsets[1:] - offsets[:-1]
    for got, want, size, d, what in ((C().expert_products(x.to(DEV), w.to(DEV), routes), y, ya, d_in, "y"), (gx, dx, dxa, d_out, "dx"),
                                     (gw, dw, dwa, max(1, int(counts.max())), "dw")):
        got, big = got.cpu(), torch.finfo(dtype).max
        plain = size <= big / 2  # (beyond it a sum on the way may pass the type's largest)
        odd = ~torch.isfinite(want)
        assert torch.equal(torch.isnan(got) & odd, torch.isnan(want)), what
        inf = torch.isinf(want)
        assert torch.equal(got.double()[inf], want[inf]), what
        assert torch.isfinite(got[plain]).all(), what
        z = torch.zeros_like(want)
        err = torch.where(plain, (got.double() - want).abs(), z)
        tol = 2 * d * 2.0 ** -23 * size + 1.001 * HALF_STEP[dtype] * want.abs() + (2.0 ** -24 if dtype == torch.float16 else 0)
        assert (err <= torch.where(plain, tol, z)).all(), what


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_products_of_a_plan_that_holds_nonsense(dtype):
    """Entries out of range are read as rows of no expert and never followed."""
    N, k, K, d = 40, 2, 4, 64
    x, w = torch.randn(N, d, device=DEV).to(dtype), torch.randn(K, d, d, device=DEV).to(dtype)
    y = torch.randn(N * k, d, device=DEV).to(dtype)
    wt = torch.rand(N, k, device=DEV)
    big = (1 << 31) - 1
    for off in ([0, 100, 7, -5, big], [-9, -8, -7, -6, -5], [big] * 5, [0, 0, 0, 0, 0]):
        for fill in (big, -big - 1, N * k):
            r = C().Routes(torch.full((N * k,), fill, dtype=torch.int32, device=DEV), torch.tensor(off, dtype=torch.int32, device=DEV),
                           torch.full((N, k), fill, dtype=torch.int32, device=DEV))
            assert (C().expert_products(x, w, r) == 0).all()
            gx, gw = C().expert_products_backward(y, x, w, r)
            assert (gx == 0).all() and (gw == 0).all()
            assert (C().combine_experts(y, wt, r) == 0).all()
            assert (C().combine_experts_backward(x, y, wt, r)[0] == 0).all()
    torch.cuda.synchronize()


def test_products_read_strided_and_unaligned_inputs():
    N, k, K, d_in, d_out = 70, 2, 4, 64, 72
    for dtype in TYPES:
        routes = C().group_routes(plan(N, k, K, 4).to(DEV), K)
        xs, ws = torch.randn(N, d_in + 9, device=DEV).to(dtype), torch.randn(K, d_out, d_in + 3, device=DEV).to(dtype)
        flat = torch.randn(N * d_in + 1, device=DEV).to(dtype)
        gs = torch.randn(d_out, N * k, device=DEV).to(dtype).t()
        w = ws[:, :, 1:d_in + 1]
        for x in (xs[:, 5:d_in + 5], flat[1:].view(N, d_in)):
            a = C().expert_products(x, w, routes)
            b = C().expert_products(x.clone(memory_format=torch.contiguous_format), w.contiguous().clone(), routes)
            assert torch.equal(a, b)
            ga, gb = (C().expert_products_backward(gs if i == 0 else gs.contiguous(), x, w, routes) for i in range(2))
            assert torch.equal(ga[0], gb[0]) and torch.equal(ga[1], gb[1])


# ------------------------------------------------------------------------------ the join
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,k,d", [(1, 1, 1), (5, 3, 7), (40, 2, 64), (33, 8, 1000), (17, 4, 2050), (3, 32, 4100), (900, 2, 12)])
def test_combine_and_gradients(N, k, d, dtype):
    K = max(k, 6)
    y = torch.randn(N * k, d, generator=gen(1)).to(dtype)
    w = torch.randn(N, k, generator=gen(2))
    g = torch.randn(N, d, generator=gen(3)).to(dtype)
    routes = C().group_routes(plan(N, k, K, N).to(DEV), K)
    pos, n_live = routes.position.cpu(), int(routes.offsets[-1])
    yd = y.to(DEV)
    yd[n_live:] = float("nan")  # rows of no expert may hold anything, weights of such slots too
    wd = torch.where(pos >= 0, w, torch.full_like(w, float("nan"))).to(DEV)
    out, size, dy, dw, dwa = ref.combine(y, w, pos, g)
    got = C().combine_experts(yd, wd, routes)
    assert got.dtype == dtype
    assert ((got.double().cpu() - out).abs() <= (k + 1) * 2.0 ** -24 * size + HALF_STEP[dtype] * out.abs() * 1.001 + 2.0 ** -24 * (dtype == torch.float16)).all()
    gy, gw = C().combine_experts_backward(g.to(DEV), yd, wd, routes)
    assert gy.dtype == dtype and gw.dtype == torch.float32
    dy[n_live:] = 0
    assert ((gy.double().cpu() - dy).abs() <= (2.0 ** -24 + HALF_STEP[dtype]) * dy.abs() * 1.001 + 2.0 ** -24 * (dtype == torch.float16)).all()
    assert ((gw.double().cpu() - dw).abs() <= (d / 32 + 8) * 2.0 ** -24 * 2 * dwa).all()
    assert (gw.cpu()[pos < 0] == 0).all()


def test_combine_reads_strided_inputs():
    N, k, d = 30, 2, 48
    routes = C().group_routes(plan(N, k, 5, 1).to(DEV), 5)
    y, w, g = torch.randn(N * k, 2 * d, device=DEV)[:, 1:2 * d:2], torch.rand(k, N, device=DEV).t(), torch.randn(N, d + 1, device=DEV)[:, 1:]
    assert torch.equal(C().combine_experts(y, w, routes), C().combine_experts(y.contiguous(), w.contiguous(), routes))
    for a, b in zip(C().combine_experts_backward(g, y, w, routes), C().combine_experts_backward(g.contiguous(), y.contiguous(), w.contiguous(), routes)):
        assert torch.equal(a, b)


# --------------------------------------------------------------------------- all together
def layer(x, router, weight, k, **kw):
    w, idx = C().route_experts(x @ router, k, **kw)
    routes = C().group_routes(idx, weight.shape[0])
    return C().combine_experts(C().expert_products(x, weight, routes), w, routes), idx


def layer64(x, router, weight, idx, func, renorm):
    x, router, weight = (t.detach().double().cpu().requires_grad_() for t in (x, router, weight))
    w = ref.weights_of(x @ router, idx.cpu(), func, renorm, 1.0)
    per = torch.einsum("nd,ked->nke", x, weight)
    out = (per.gather(1, idx.cpu().long()[:, :, None].expand(-1, -1, per.shape[2])) * w[:, :, None]).sum(1)
    return out, (x, router, weight)


@pytest.mark.parametrize("func,renorm", [("softmax", True), ("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_layer_and_its_gradients(func, renorm):
    """The operators together, forward and through autograd, against the same layer in 64 bits (fp32: 1e-5 of the
    largest entry covers sums of 64 to 200 terms at 2^-23 each with a factor of ten to spare)."""
    N, K, k, d_in, d_out = 200, 8, 2, 64, 48
    x, router = torch.randn(N, d_in, device=DEV).requires_grad_(), (torch.randn(d_in, K, device=DEV) / 8).requires_grad_()
    weight = (torch.randn(K, d_out, d_in, device=DEV) / 8).requires_grad_()
    out, idx = layer(x, router, weight, k, score_func=func, renormalize=renorm)
    g = torch.randn(N, d_out, device=DEV)
    out.backward(g)
    want, leaves = layer64(x, router, weight, idx, func, renorm)
    want.backward(g.double().cpu())
    for a, b in [(out, want)] + [(p.grad, q.grad) for p, q in zip((x, router, weight), leaves)]:
        a, b = a.detach().double().cpu(), b.detach()
        assert float((a - b).abs().max()) <= 1e-5 * float(b.abs().max())
    with torch.no_grad():
        assert torch.equal(layer(x, router, weight, k, score_func=func, renormalize=renorm)[0], out)


def test_layer_gradient_of_some_inputs_only():
    x, router, weight = torch.randn(30, 16, device=DEV), torch.randn(16, 4, device=DEV), torch.randn(4, 8, 16, device=DEV)
    whole = [t.clone().requires_grad_() for t in (x, router, weight)]
    layer(*whole, 2)[0].sum().backward()
    for i in range(3):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, router, weight))]
        layer(*some, 2)[0].sum().backward()
        assert torch.equal(some[i].grad, whole[i].grad)
    # a broadcast gradient (of sum()) and an integer output that takes none
    w, idx = C().route_experts((x @ router).requires_grad_(), 2)
    assert w.requires_grad and not idx.requires_grad


def test_two_products_one_after_the_other():
    """Grouped rows as points of one slot each: their plan is the identity, and the layer of two products has its gradients."""
    N, k, K, d, hidden = 60, 2, 5, 24, 40
    x, w1, w2 = (torch.randn(*s, generator=gen(i)).to(DEV).requires_grad_() for i, s in enumerate(((N, d), (K, hidden, d), (K, d, hidden))))
    idx, wt = plan(N, k, K, 9).to(DEV), torch.rand(N, k, generator=gen(5)).to(DEV)
    routes = C().group_routes(idx, K)
    same = C().group_routes(idx.flatten()[routes.order.long()][:, None].contiguous(), K)
    live = int(routes.offsets[-1])
    assert torch.equal(same.order, torch.arange(N * k, dtype=torch.int32, device=DEV)) and torch.equal(same.offsets, routes.offsets)
    assert torch.equal(same.position[:live, 0], same.order[:live]) and (same.position[live:] == -1).all()
    h = torch.nn.functional.silu(C().expert_products(x, w1, routes))
    out = C().combine_experts(C().expert_products(h, w2, same), wt, routes)
    grads = torch.autograd.grad(out.sum(), (x, w1, w2))
    x64, w164, w264 = (t.detach().double().requires_grad_() for t in (x, w1, w2))
    e = idx.long().clamp(min=0)
    h64 = torch.nn.functional.silu(torch.einsum("nd,nkhd->nkh", x64, w164[e]))
    out64 = (torch.einsum("nkh,nkdh->nkd", h64, w264[e]) * (wt.double() * (idx >= 0))[:, :, None]).sum(1)
    want = torch.autograd.grad(out64.sum(), (x64, w164, w264))
    # (sums of at most N k + d + hidden fp32 terms in a row)
    for got, exact in zip((out.detach(), *grads), (out64.detach(), *want)):
        assert float((got.double() - exact).abs().max()) <= 2 * (N * k + d + hidden) * 2.0 ** -23 * float(exact.abs().max())


def test_no_points():
    z = torch.empty(0, 8, device=DEV)
    w, idx = C().route_experts(z, 2)
    assert w.shape == (0, 2) and idx.shape == (0, 2)
    assert C().route_experts_backward(w, z, idx).shape == (0, 8)
    routes = C().group_routes(idx, 8)
    assert (routes.offsets == 0).all() and routes.order.numel() == 0 and routes.position.shape == (0, 2)
    x, weight = torch.empty(0, 16, device=DEV), torch.randn(8, 4, 16, device=DEV)
    y = C().expert_products(x, weight, routes)
    assert y.shape == (0, 4)
    gx, gw = C().expert_products_backward(y, x, weight, routes)
    assert gx.shape == (0, 16) and (gw == 0).all() and gw.shape == weight.shape
    out = C().combine_experts(y, w, routes)
    assert out.shape == (0, 4)
    gy, gww = C().combine_experts_backward(out, y, w, routes)
    assert gy.shape == (0, 4) and gww.shape == (0, 2)


def test_same_results_every_time():
    x, router, weight = torch.randn(3000, 64, device=DEV), torch.randn(64, 16, device=DEV), torch.randn(16, 96, 64, device=DEV)
    for dtype in TYPES:
        args = [t.to(dtype) for t in (x, router, weight)]
        first = [t.clone().requires_grad_() for t in args]
        a = layer(*first, 3)[0]
        a.float().square().sum().backward()
        for _ in range(3):
            again = [t.clone().requires_grad_() for t in args]
            b = layer(*again, 3)[0]
            b.float().square().sum().backward()
            assert torch.equal(a, b) and all(torch.equal(p.grad, q.grad) for p, q in zip(first, again))


def test_on_another_stream():
    x, router, weight = torch.randn(500, 64, device=DEV), torch.randn(64, 16, device=DEV), torch.randn(16, 96, 64, device=DEV)
    want = layer(x, router, weight, 2)[0]
    torch.cuda.synchronize()
    s, t = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(5):  # two streams at once
        for stream in (s, t):
            with torch.cuda.stream(stream):
                outs.append(layer(x, router, weight, 2)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def capture(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        graphs.append((graph, outs))
    return graphs


def replay_both(graphs, step, x):
    """Two graphs of the same calls, replayed in turn on new inputs."""
    for seed in (1, 2):
        x.copy_(torch.randn(x.shape, generator=gen(seed)))
        for graph, outs in graphs:
            graph.replay()
        torch.cuda.synchronize()
        want = step()
        for _, outs in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("dtype", TYPES)
def test_captured_and_replayed(dtype):
    """The backward functions are captured while an eager graph of the same leaves lives."""
    N, K = 300, 8
    x = torch.randn(N, 64, device=DEV).to(dtype)
    router = torch.randn(64, K, device=DEV).to(dtype).requires_grad_()
    weight = torch.randn(K, 48, 64, device=DEV).to(dtype).requires_grad_()
    eager = layer(x, router, weight, 2)[0]

    def step():
        with torch.no_grad():
            z = x @ router
            w, idx = C().route_experts(z, 2)
            routes = C().group_routes(idx, K)
            y = C().expert_products(x, weight, routes)
            out = C().combine_experts(y, w, routes)
            gy, gw = C().combine_experts_backward(2 * out, y, w, routes)
            return [out, *C().expert_products_backward(gy, x, weight, routes), C().route_experts_backward(gw, z, idx)]
    replay_both(capture(step), step, x)
    assert eager.requires_grad


def test_autograd_captured_and_replayed():
    N, K = 300, 8
    x = torch.randn(N, 64, device=DEV)
    router = torch.randn(64, K, device=DEV).requires_grad_()
    weight = torch.randn(K, 48, 64, device=DEV).requires_grad_()

    def step():
        out = layer(x, router, weight, 2)[0]
        return [out.detach(), *torch.autograd.grad(out.square().sum(), (router, weight))]
    replay_both(capture(step), step, x)


def test_gpu_refusals():
    z = torch.randn(6, 8, device=DEV)
    w, idx = C().route_experts(z, 2)
    routes = C().group_routes(idx, 8)
    x, weight = torch.randn(6, 16, device=DEV), torch.randn(8, 4, 16, device=DEV)
    y = C().expert_products(x, weight, routes)
    bad = [lambda: C().route_experts(z, 0), lambda: C().route_experts(z, 9), lambda: C().route_experts(z[0], 2),
           lambda: C().route_experts(z, 2, n_groups=3), lambda: C().route_experts(z, 2, n_groups=4, top_groups=5),
           lambda: C().route_experts(z, 2, bias=torch.zeros(7, device=DEV)), lambda: C().route_experts(z, 2, bias=torch.zeros(8)),
           lambda: C().route_experts(z, 2, bias=torch.zeros(8, device=DEV).bfloat16()),
           lambda: C().route_experts(torch.randn(2, 4097, device=DEV), 2), lambda: C().route_experts(torch.empty(2, 0, device=DEV), 1),
           lambda: C().route_experts_backward(w.bfloat16(), z, idx), lambda: C().route_experts_backward(w[:3], z, idx),
           lambda: C().route_experts_backward(w, z, idx.long()), lambda: C().group_routes(idx[0], 8), lambda: C().group_routes(idx, 0),
           lambda: C().group_routes(idx, 4097), lambda: C().expert_products(x, weight.bfloat16(), routes),
           lambda: C().expert_products(x[:5], weight, routes), lambda: C().expert_products(x, weight[:7], routes),
           lambda: C().expert_products(x, weight[:, :, :15], routes), lambda: C().expert_products(x, weight, routes._replace(order=routes.order[:-1])),
           lambda: C().expert_products(x, weight, routes._replace(offsets=routes.offsets.cpu())),
           lambda: C().expert_products(x, weight, routes._replace(position=routes.position.long())),
           lambda: C().expert_products_backward(y[:-1], x, weight, routes), lambda: C().expert_products_backward(y.half(), x, weight, routes),
           lambda: C().combine_experts(y[:-1], w, routes), lambda: C().combine_experts(y, w.half(), routes),
           lambda: C().combine_experts(y, w[:, :1], routes), lambda: C().combine_experts_backward(x, y, w, routes)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()


# ---------------------------------------------------------------------------- the models
@pytest.mark.parametrize("model", ["NativeFlashGMM", "NativeStandardGMM"])
def test_models_route_by_their_responsibilities(model):
    from flashgmm_b200 import native_wrapper
    from flashgmm_b200.data import make_mixture
    N, K, d, k, d_out = 1500, 12, 16, 3, 10
    X = make_mixture(N, K, d, seed=3)[0].to(DEV)
    m = getattr(native_wrapper, model)(K, d, max_iter=5)
    m.fit(X)
    gamma = m.predict_proba(X)
    w, idx = m.route(X, k)
    want = ref.route(gamma.cpu(), k, "given")
    check_route(gamma, (w, idx), want, "given", 1.0)
    assert torch.equal(idx[:, 0].long(), m.predict(X))
    raw = m.route(X, k, renormalize=False)[0]
    assert torch.equal(raw, gamma.gather(1, idx.long()))
    weight = torch.randn(K, d_out, d, device=DEV).requires_grad_()
    out = m.mix_experts(X, weight, k)
    per = torch.einsum("nd,ked->nke", X.double(), weight.detach().double())
    exact = (per.gather(1, idx.long()[:, :, None].expand(-1, -1, d_out)) * w.double()[:, :, None]).sum(1)
    assert float((out.detach().double() - exact).abs().max()) <= 1e-5 * float(exact.abs().max())
    out.sum().backward()
    assert weight.grad.shape == weight.shape and torch.isfinite(weight.grad).all()


def test_model_experts_pass_gradients_to_the_points():
    from flashgmm_b200 import native_wrapper
    from flashgmm_b200.data import make_mixture
    N, K, d, k, d_out = 400, 6, 12, 2, 20
    X = make_mixture(N, K, d, seed=5)[0].to(DEV)
    m = native_wrapper.NativeFlashGMM(K, d, max_iter=3)
    m.fit(X)
    w, idx = m.route(X, k)
    weight = torch.randn(K, d_out, d, device=DEV)
    points = X.clone().requires_grad_()
    grad, = torch.autograd.grad(m.mix_experts(points, weight, k).sum(), points)
    exact = (weight.double().sum(1)[idx.long()] * w.double()[:, :, None]).sum(1)  # the gate has no gradient
    size = (weight.double().abs().sum(1)[idx.long()] * w.double()[:, :, None]).sum(1)
    assert ((grad.double() - exact).abs() <= 2 * (d_out + k) * 2.0 ** -23 * size).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_products_of_many_rows(dtype):
    """Enough rows and columns for the widest tiles in each direction (results in 64 bits on the GPU)."""
    N, k, K, d_in, d_out = 3000, 4, 8, 1032, 1040
    g = torch.Generator(device=DEV).manual_seed(1)
    x, w = torch.randn(N, d_in, generator=g, device=DEV).to(dtype), (torch.randn(K, d_out, d_in, generator=g, device=DEV) / 32).to(dtype)
    dy = torch.randn(N * k, d_out, generator=g, device=DEV).to(dtype)
    routes = C().group_routes(plan(N, k, K, 2).to(DEV), K)
    y, ya, dx, dxa, dw, dwa = ref.products(x, w, routes.order, routes.offsets, k, dy)
    close(C().expert_products(x, w, routes), y.cpu(), ya.cpu(), d_in, dtype, "y")
    gx, gw = C().expert_products_backward(dy, x, w, routes)
    close(gx, dx.cpu(), dxa.cpu(), d_out + k, dtype, "dx")
    counts = routes.offsets[1:] - routes.offsets[:-1]
    close(gw, dw.cpu(), dwa.cpu(), int(counts.max()), dtype, "dw")
