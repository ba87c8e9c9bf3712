"""Tensors that the expert operators do not read through their pointers are refused before anything is launched."""
import pytest
import torch
import torch.autograd.forward_ad as fw
from torch._subclasses.fake_tensor import FakeTensorMode

from flashgmm_b200 import flash_gmm_native as C


def calls():
    """Each operator with each of its floating-point inputs in turn: (call, that input)."""
    z, x, w, y, wt = torch.randn(3, 4), torch.randn(3, 6), torch.randn(4, 5, 6), torch.randn(6, 5), torch.rand(3, 2)
    g, idx = torch.randn(3, 5), torch.zeros(3, 2, dtype=torch.int32)
    routes = C.Routes(torch.zeros(6, dtype=torch.int32), torch.zeros(5, dtype=torch.int32), idx)
    return [(lambda t: C.route_experts(t, 2), z), (lambda t: C.route_experts_backward(wt, t, idx), z),
            (lambda t: C.expert_products(t, w, routes), x), (lambda t: C.expert_products_backward(y, t, w, routes), x),
            (lambda t: C.combine_experts(t, wt, routes), y), (lambda t: C.combine_experts_backward(g, t, wt, routes), y)]


@pytest.mark.parametrize("i", range(6))
def test_forward_mode_is_refused(i):
    call, t = calls()[i]
    with fw.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        call(fw.make_dual(t, torch.ones_like(t)))


@pytest.mark.parametrize("i", range(6))
def test_traced_batched_and_sparse_tensors_are_refused(i):
    call, t = calls()[i]
    with FakeTensorMode(allow_non_fake_inputs=True):
        traced = torch.empty(t.shape[0] + 1, *t.shape[1:], device="cuda", dtype=t.dtype)
        with pytest.raises(RuntimeError, match="plain"):
            call(traced[1:])  # (its pointer would be a few bytes above zero)
    with pytest.raises(RuntimeError, match="plain"):
        torch.func.vmap(call)(t[None].clone())
    with pytest.raises(RuntimeError, match="plain"):
        torch.func.jvp(call, (t,), (torch.ones_like(t),))
    with pytest.raises(RuntimeError, match="plain"):
        call(t.to_sparse())
