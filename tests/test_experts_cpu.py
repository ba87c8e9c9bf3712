"""The expert operators without a GPU: refusals of the Python entry points and of the C ABI (whose checks come
before any launch), and their workspace queries."""
import ctypes

import pytest
import torch

from flashgmm_b200 import _lib
from flashgmm_b200 import flash_gmm_native as C

P = ctypes.c_void_p(4096)  # stands for a device pointer; the checks come before any use


def test_entry_points_are_exported():
    import flash_gmm_native as top
    for name in ("Routes", "route_experts", "route_experts_backward", "group_routes", "expert_products",
                 "expert_products_backward", "combine_experts", "combine_experts_backward"):
        assert name in C.__all__ and getattr(C, name) is getattr(top, name)


def test_python_refuses_what_is_no_cuda_tensor():
    z = torch.randn(3, 4)
    routes = C.Routes(torch.zeros(6, dtype=torch.int32), torch.zeros(5, dtype=torch.int32),
                      torch.zeros(3, 2, dtype=torch.int32))
    for call in (lambda: C.route_experts(z, 2), lambda: C.route_experts_backward(z[:, :2], z, routes.position),
                 lambda: C.group_routes(routes.position, 4), lambda: C.expert_products(z, torch.randn(4, 5, 4), routes),
                 lambda: C.expert_products_backward(torch.randn(6, 5), z, torch.randn(4, 5, 4), routes),
                 lambda: C.combine_experts(torch.randn(6, 5), z[:, :2], routes),
                 lambda: C.combine_experts_backward(z, torch.randn(6, 4), z[:, :2], routes)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_python_refuses_other_types():
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        C.route_experts(torch.randn(3, 4).double(), 2)
    with pytest.raises(RuntimeError, match="torch.Tensor"):
        C.route_experts([[1.0, 2.0]], 1)
    with pytest.raises(RuntimeError, match="score_func"):
        C.route_experts(torch.randn(3, 4), 2, score_func="tanh")
    with pytest.raises(RuntimeError, match="Int"):
        C.group_routes(torch.zeros(3, 2, dtype=torch.int64), 4)
    with pytest.raises(RuntimeError, match="Routes"):
        C.expert_products(torch.randn(3, 4), torch.randn(4, 5, 4), (1, 2, 3))


def _route(dtype=0, N=4, K=8, stride=8, top_k=2, func=0, n_groups=1, top_groups=1, z=P, w=P, i=P):
    return _lib.load().fgmm_route_experts(z, dtype, N, K, stride, None, top_k, func, n_groups, top_groups, 1, 1.0, w, i, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=3), 1), (dict(N=-1), 1), (dict(K=0), 1), (dict(top_k=0), 1), (dict(top_k=9), 1), (dict(func=3), 1),
    (dict(n_groups=3), 1), (dict(n_groups=0), 1), (dict(n_groups=2, top_groups=3), 1), (dict(n_groups=2, top_groups=0), 1),
    (dict(stride=-8), 1), (dict(K=4097, stride=4097), 2), (dict(K=64, top_k=33), 1), (dict(N=1 << 31), 2), (dict(N=(1 << 30) - 512), 2),
    (dict(z=None), 1), (dict(w=None), 1), (dict(i=None), 1), (dict(z=ctypes.c_void_p(4098)), 1),
    (dict(K=64, n_groups=64), 1)])
def test_route_refusals(kw, code):
    assert _route(**kw) == code
    assert _lib.load().fgmm_last_error()


def test_no_points_is_no_work():
    assert _route(N=0, z=None, w=None, i=None) == 0
    lib = _lib.load()
    assert lib.fgmm_expert_products(None, 0, 0, 4, None, 4, 4, None, None, 2, None, None, 0, None) == 0
    assert lib.fgmm_combine_experts(None, 0, 0, 4, None, None, 2, None, None) == 0
    assert lib.fgmm_combine_experts_backward(None, None, 0, 0, 4, None, None, None, 4, 2, None, None, None) == 0


def test_group_refusals_and_workspace():
    lib = _lib.load()
    assert lib.fgmm_group_routes_workspace_bytes(-1, 4) == 0
    assert lib.fgmm_group_routes_workspace_bytes(10, 0) == 0
    assert lib.fgmm_group_routes_workspace_bytes(10, 4097) == 0
    need = lib.fgmm_group_routes_workspace_bytes(5000, 64)
    assert need > 0
    assert lib.fgmm_group_routes(P, 5000, 64, P, P, P, P, need - 1, None) == _lib.FGMM_ERR_WORKSPACE
    assert lib.fgmm_group_routes(P, 5000, 64, P, P, P, ctypes.c_void_p(4097), need, None) == _lib.FGMM_ERR_INVALID
    assert lib.fgmm_group_routes(None, 5000, 64, P, P, P, P, need, None) == _lib.FGMM_ERR_INVALID
    assert lib.fgmm_group_routes(P, 5000, 4097, P, P, P, P, need, None) == _lib.FGMM_ERR_UNSUPPORTED


def test_products_refusals():
    lib = _lib.load()
    need = lib.fgmm_expert_products_workspace_bytes(1, 16, 8, 32, 64, 2)
    assert need > 0

    def call(dtype=1, N=16, d_in=32, K=8, d_out=64, top_k=2, x=P, w=P, order=P, off=P, y=P, ws=P, nb=need):
        return lib.fgmm_expert_products(x, dtype, N, d_in, w, K, d_out, order, off, top_k, y, ws, nb, None)
    for kw, code in ((dict(dtype=7), 1), (dict(d_in=0), 1), (dict(d_out=0), 1), (dict(K=5000), 2), (dict(top_k=0), 1),
                     (dict(x=None), 1), (dict(w=None), 1), (dict(order=None), 1), (dict(off=None), 1), (dict(y=None), 1),
                     (dict(ws=None), 1), (dict(nb=need - 1), 3), (dict(x=ctypes.c_void_p(4097)), 1),
                     (dict(N=1 << 30, top_k=2), 2), (dict(d_in=(1 << 20) + 1), 2)):
        assert call(**kw) == code, kw
    back = lib.fgmm_expert_products_backward_workspace_bytes(1, 16, 8, 32, 64, 2)
    assert back >= 16 * 2 * 32 * 2

    def backward(dy=P, x=P, w=P, pos=P, dx=P, dw=P, nb=back):
        return lib.fgmm_expert_products_backward(dy, x, 1, 16, 32, w, 8, 64, P, P, pos, 2, dx, dw, P, nb, None)
    assert backward(dy=None) == 1 and backward(x=None) == 1 and backward(w=None) == 1 and backward(pos=None) == 1
    assert backward(nb=back - 1) == 3


def test_workspaces_of_no_points():
    lib = _lib.load()
    for dtype in (0, 1, 2):
        assert lib.fgmm_expert_products_workspace_bytes(dtype, 0, 8, 32, 64, 2) > 0
        assert lib.fgmm_expert_products_backward_workspace_bytes(dtype, 0, 8, 32, 64, 2) > 0


def test_combine_refusals():
    lib = _lib.load()
    assert lib.fgmm_combine_experts(P, 5, 4, 8, P, P, 2, P, None) == 1
    assert lib.fgmm_combine_experts(P, 0, 4, 0, P, P, 2, P, None) == 1
    assert lib.fgmm_combine_experts(P, 0, 4, 8, None, P, 2, P, None) == 1
    assert lib.fgmm_combine_experts(ctypes.c_void_p(4098), 0, 4, 8, P, P, 2, P, None) == 1
    assert lib.fgmm_combine_experts_backward(P, P, 0, 4, 8, P, None, P, 8, 2, P, P, None) == 1
    assert lib.fgmm_combine_experts_backward(P, P, 0, 4, 8, P, P, P, 0, 2, P, P, None) == 1
