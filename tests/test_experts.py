"""Rows that go to experts without a GPU: what the entry points refuse."""
import numpy as np
import pytest
import torch

from permutohedral_encoding_amd import _native, layers


def _memory():
    block = np.zeros(4096, np.uint8)
    return block, block.ctypes.data + (-block.ctypes.data) % 64


def test_the_entry_points_refuse_before_they_launch():
    lib = _native.lib()
    block, p = _memory()
    z = None
    assert lib.penc_route(3, 4, 8, 2, 1, p, 8, p, p, z) == 10
    for bad in ((-1, 8, 2), (1 << 31, 8, 2), (4, 0, 1), (4, 1025, 1), (4, 8, 0), (4, 8, 9), (4, 1, 2), (1 << 30, 8, 2)):
        assert lib.penc_route(0, *bad, 1, p, 8, p, p, z) == 12 == lib.penc_route_backward(0, *bad, 1, p, 8, p, p, p, p, z)
    assert lib.penc_route(0, 4, 8, 2, 1, p, -1, p, p, z) == 12
    assert lib.penc_route(0, 4, 8, 2, 1, z, 8, p, p, z) == 1 and lib.penc_route(0, 4, 8, 2, 1, p, 8, z, p, z) == 1 and lib.penc_route(0, 4, 8, 2, 1, p, 8, p, z, z) == 1
    assert lib.penc_route(1, 4, 8, 2, 1, p + 1, 8, p, p, z) == 5 and lib.penc_route(0, 4, 8, 2, 1, p, 8, p + 2, p, z) == 5
    assert lib.penc_route(0, 0, 8, 2, 1, z, 8, z, z, z) == 0
    assert lib.penc_route_backward(0, 4, 8, 2, 0, z, 8, p, p, p, p, z) == 1 and lib.penc_route_backward(0, 4, 8, 2, 1, z, 8, p, p, z, p, z) == 1
    # plans: a few choices need no workspace
    assert lib.penc_plan_workspace_bytes(16384, 8) == 0 == lib.penc_plan_workspace_bytes(-1, 8) == lib.penc_plan_workspace_bytes(10000, 1025)
    need = lib.penc_plan_workspace_bytes(20000, 8)
    assert need == 4 * 9 * (20 + 1)
    assert lib.penc_plan(2, 10, 8, p, p, p, z, 0, z) == 10 and lib.penc_plan(4, -1, 8, p, p, p, z, 0, z) == 12 and lib.penc_plan(4, 10, 0, p, p, p, z, 0, z) == 12
    assert lib.penc_plan(4, 10, 8, z, p, p, z, 0, z) == 1 and lib.penc_plan(4, 10, 8, p, p, z, z, 0, z) == 1 and lib.penc_plan(8, 10, 8, p + 4, p, p, z, 0, z) == 5
    assert lib.penc_plan(4, 20000, 8, p, p, p, p, need - 1, z) == 8 and lib.penc_plan(4, 20000, 8, p, p, p, z, need, z) == 1
    # rows there and back
    assert lib.penc_dispatch(3, 4, 2, 8, p, 8, p, p, p, z) == 10
    for bad in ((-1, 2, 8), (4, 0, 8), (4, 1025, 8), (4, 2, 0), (4, 2, (1 << 24) + 1), (1 << 30, 2, 8)):
        assert lib.penc_dispatch(0, *bad, p, 8, p, p, p, z) == 12 == lib.penc_combine(0, 0, *bad, p, 8, p, p, p, p, z)
        assert lib.penc_combine_backward(0, 0, *bad, p, 8, p, 8, p, p, p, p, p, z) == 12
    assert lib.penc_dispatch(0, 4, 2, 8, z, 8, p, p, p, z) == 1 and lib.penc_dispatch(0, 4, 2, 8, p, 8, z, p, p, z) == 1 and lib.penc_dispatch(0, 4, 2, 8, p, 8, p, z, p, z) == 1
    assert lib.penc_dispatch(0, 4, 2, 8, p + 2, 8, p, p, p, z) == 5 and lib.penc_dispatch(1, 0, 2, 8, z, 8, z, z, z, z) == 0
    assert lib.penc_combine(1, 2, 4, 2, 8, p, 8, p, p, p, p, z) == 10 and lib.penc_combine(1, 1, 4, 2, 8, p, 8, p + 1, p, p, p, z) == 5
    assert lib.penc_combine(0, 0, 4, 2, 8, z, 8, p, p, p, p, z) == 1
    assert lib.penc_combine_backward(0, 0, 4, 2, 8, p, 8, z, 8, p, p, p, z, p, z) == 1  # the weights' gradient needs y
    assert lib.penc_combine_backward(0, 0, 4, 2, 8, p, 8, z, 8, p, p, p, z, z, z) == 0  # nothing is wanted


def test_the_products_refuse_before_they_launch():
    lib = _native.lib()
    block, p = _memory()
    z = None
    assert lib.penc_expert_linear(3, 4, 2, 8, 8, p, 8, p, p, p, p, z) == 10 == lib.penc_expert_linear_input_grad(-1, 4, 2, 8, 8, p, 8, p, p, p, z)
    assert lib.penc_expert_weight_grad(7, 4, 2, 8, 8, p, 8, p, 8, p, p, p, p, 0, z) == 10
    for bad in ((-1, 2, 8, 8), (1 << 31, 2, 8, 8), (4, 0, 8, 8), (4, 1025, 8, 8), (4, 2, 0, 8), (4, 2, 8, 0), (4, 2, (1 << 18) + 1, 8), (4, 2, 8, (1 << 18) + 1)):
        assert lib.penc_expert_linear(0, *bad, p, 1 << 19, p, p, p, p, z) == 12 == lib.penc_expert_linear_input_grad(0, *bad, p, 1 << 19, p, p, p, z)
        assert lib.penc_expert_weight_grad(0, *bad, p, 1 << 19, p, 1 << 19, p, p, p, p, 0, z) == 12 and lib.penc_expert_weight_grad_workspace_bytes(0, *bad) == 0
    # rows that overlap, and rows too far apart
    for stride in (7, -8, (1 << 20) + 1):
        assert lib.penc_expert_linear(0, 4, 2, 8, 8, p, stride, p, p, p, p, z) == 12 == lib.penc_expert_linear_input_grad(0, 4, 2, 8, 8, p, stride, p, p, p, z)
        assert lib.penc_expert_weight_grad(0, 4, 2, 8, 8, p, 8, p, stride, p, p, p, p, 0, z) == 12 == lib.penc_expert_weight_grad(0, 4, 2, 8, 8, p, stride, p, 8, p, p, p, p, 0, z)
    assert lib.penc_expert_linear(0, 4, 2, 8, 8, z, 8, p, p, p, p, z) == 1 == lib.penc_expert_linear(0, 4, 2, 8, 8, p, 8, p, p, z, p, z)
    assert lib.penc_expert_linear(0, 4, 2, 8, 8, p + 2, 8, p, p, p, p, z) == 5 and lib.penc_expert_linear(1, 4, 2, 8, 8, p, 8, p, p + 1, p, p, z) == 5
    assert lib.penc_expert_linear(0, 0, 2, 8, 8, z, 8, z, z, z, z, z) == 0 == lib.penc_expert_linear_input_grad(0, 0, 2, 8, 8, z, 8, z, z, z, z)
    need = lib.penc_expert_weight_grad_workspace_bytes(0, 1 << 20, 8, 64, 64)
    assert 4 * 65 * 64 * 8 < need < 1 << 26 and lib.penc_expert_weight_grad_workspace_bytes(0, 100, 8, 64, 64) == 0
    assert lib.penc_expert_weight_grad(0, 1 << 20, 8, 64, 64, p, 64, p, 64, p, p, p, p, need - 1, z) == 8
    assert lib.penc_expert_weight_grad(0, 1 << 20, 8, 64, 64, p, 64, p, 64, p, p, p, z, need, z) == 1
    assert lib.penc_expert_weight_grad(0, 4, 8, 64, 64, p, 64, p, 64, p, z, p, p, need, z) == 1


def test_all_gradients_refuse_before_they_launch():
    lib = _native.lib()
    block, p = _memory()
    z = None
    assert lib.penc_expert_linear_grads(7, 4, 2, 8, 8, p, 8, p, 8, p, p, p, p, p, p, 0, z) == 10
    for bad in ((-1, 2, 8, 8), (1 << 31, 2, 8, 8), (4, 0, 8, 8), (4, 1025, 8, 8), (4, 2, 0, 8), (4, 2, 8, 0), (4, 2, (1 << 18) + 1, 8), (4, 2, 8, (1 << 18) + 1)):
        assert lib.penc_expert_linear_grads(0, *bad, p, 1 << 19, p, 1 << 19, p, p, p, p, p, p, 0, z) == 12
    for stride in (7, -8, (1 << 20) + 1):
        assert lib.penc_expert_linear_grads(0, 4, 2, 8, 8, p, 8, p, stride, p, p, p, p, p, p, 0, z) == 12
        assert lib.penc_expert_linear_grads(0, 4, 2, 8, 8, p, stride, p, 8, p, p, p, p, p, p, 0, z) == 12
    for k in (0, 1, 2, 3, 5):  # x, the gradient, the weight (where dx is wanted), the offsets and the weight's gradient
        given = [p] * 6
        given[k] = z
        x, grad, weight, offsets, dx, dweight = given
        assert lib.penc_expert_linear_grads(0, 4, 2, 8, 8, x, 8, grad, 8, weight, offsets, dx, dweight, z, z, 0, z) == 1
        given = [p] * 6
        given[k] = p + 2
        x, grad, weight, offsets, dx, dweight = given
        assert lib.penc_expert_linear_grads(0, 4, 2, 8, 8, x, 8, grad, 8, weight, offsets, dx, dweight, z, z, 0, z) == 5
    need = lib.penc_expert_weight_grad_workspace_bytes(0, 1 << 20, 8, 64, 64)
    assert lib.penc_expert_linear_grads(0, 1 << 20, 8, 64, 64, p, 64, p, 64, p, p, p, p, p, p, need - 1, z) == 8
    assert lib.penc_expert_linear_grads(0, 1 << 20, 8, 64, 64, p, 64, p, 64, p, p, p, p, p, z, need, z) == 1


def test_tensors_in_host_memory_are_refused():
    x, experts = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int64)
    plan = layers.Routing(experts, 3, experts.int(), torch.zeros(4, dtype=torch.int32))
    for call in (lambda: layers.route(x), lambda: layers.routing(experts, 3), lambda: layers.dispatch(x, plan), lambda: layers.combine(x, x, plan),
                 lambda: layers.expert_linear(x, x[None], None, plan)):
        with pytest.raises(ValueError, match="GPU memory"):
            call()


def test_orthogonalise_refuses_before_it_launches():
    lib = _native.lib()
    block, p = _memory()
    p += (-p) % 256
    z, good = None, (3.4445, -4.7750, 2.0315)
    call = lambda t=0, m=1, r=8, c=9, steps=5, k=good, eps=1e-7, g=p, to=p + 1024, ws=p, n=1 << 30: lib.penc_orthogonalise(t, m, r, c, steps, *k, eps, g, to, ws, n, z)  # noqa: E731
    assert call(t=3) == 10 and call(m=-1) == 12 and call(m=(1 << 20) + 1) == 12 and call(r=0) == 12 and call(c=(1 << 16) + 1) == 12 and call(steps=0) == 12 and call(steps=65) == 12
    assert call(eps=0.0) == 11 and call(eps=float("nan")) == 11 and call(eps=float("inf")) == 11
    # singular values over 3 and factors over 15 are refused, wherever on the way they come up
    for k in ((4.0, 0.0, 0.0), (float("nan"), 0.0, 0.0), (1.0, 16.0, -16.0), (2.0, 1.5, 0.0), (0.0, 0.0, float("inf"))):
        assert call(k=k) == 11
    assert call(k=(2.0, 0.0, 0.0), steps=1, g=z) == 1 and call(k=(2.0, 0.0, 0.0), steps=2) == 11
    assert call(k=(1.5, -0.5, 0.0), steps=64, g=z) == 1 and call(steps=64, g=z) == 1
    assert call(g=z) == 1 and call(to=z) == 1 and call(g=p + 2) == 5 and call(to=p + 4) == 5 and call(ws=p + 16) == 5 and call(m=0, g=z, to=z) == 0
    # small matrices need no workspace
    assert lib.penc_orthogonalise_workspace_bytes(0, 100, 64, 256) == 0 == lib.penc_orthogonalise_workspace_bytes(0, 1, 0, 4)
    need = lib.penc_orthogonalise_workspace_bytes(2, 2, 1000, 203)
    assert need >= 2 * (2 * 1000 * 256 + 2 * 203 * 256) * 2 and lib.penc_orthogonalise_workspace_bytes(0, 2, 1000, 203) > need
    assert call(t=2, m=2, r=1000, c=203, n=need - 1) == 8 and call(t=2, m=2, r=1000, c=203, ws=z) == 1
    assert lib.penc_muon_momentum(0, -1, p, p, 0.9, 1, p, z) == 12 and lib.penc_muon_momentum(0, 4, z, p, 0.9, 1, p, z) == 1 and lib.penc_muon_momentum(0, 0, z, z, 0.9, 1, z, z) == 0
    assert lib.penc_muon_apply(4, 4, p, p, 1.0, 0.1, z) == 10 and lib.penc_muon_apply(0, 4, p, p + 2, 1.0, 0.1, z) == 5 and lib.penc_muon_apply(0, 4, p, z, 1.0, 0.1, z) == 1
