"""Forward-mode derivatives through the mixture layer's operators are refused, not lost: a dual tensor does not require a
gradient, so nothing else would notice its tangent.  Host only: the refusal comes before the device is asked for."""

import pytest
import torch
from torch.autograd import forward_ad

from triturus_amd.gmm import gmm, gmm_grad
from triturus_amd.mx4 import MX4, mm_mx4
from triturus_amd.route import Routes, route, route_grad


def calls(dual):
    a, b, s, g = torch.randn(6, 8), torch.randn(2, 8, 4), torch.tensor([3, 3]), torch.randn(6, 4)
    q = MX4(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), 8)
    logits, ints = torch.randn(6, 5), torch.zeros(6, 2, dtype=torch.int32)
    w, gw = torch.rand(6, 2), torch.randn(6, 2)
    return {
        "gmm a": lambda: gmm(dual(a), b, s), "gmm b": lambda: gmm(a, dual(b), s),
        "gmm_grad g": lambda: gmm_grad(dual(g), a, b, s), "gmm_grad a": lambda: gmm_grad(g, dual(a), b, s), "gmm_grad b": lambda: gmm_grad(g, a, dual(b), s),
        "mm_mx4": lambda: mm_mx4(dual(a), q), "route": lambda: route(dual(logits), 2),
        "route_grad g": lambda: route_grad(dual(gw), logits, Routes(w, ints, s, ints, s)),
        "route_grad logits": lambda: route_grad(gw, dual(logits), Routes(w, ints, s, ints, s)),
        "route_grad weights": lambda: route_grad(gw, logits, Routes(dual(w), ints, s, ints, s)),
    }


@pytest.mark.parametrize("name", list(calls(None)))
def test_tangents_are_refused(name):
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))[name]()
        with pytest.raises(RuntimeError, match="forward-mode"):
            with torch.no_grad():
                calls(lambda t: forward_ad.make_dual(t, torch.ones_like(t)))[name]()
        with pytest.raises(RuntimeError, match="GPU only"):  # no tangent: as outside
            calls(lambda t: t)[name]()


def test_functional_transform_is_refused():
    a, b, s = torch.randn(6, 8), torch.randn(2, 8, 4), torch.tensor([3, 3])
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: gmm(x, b, s), (a,), (torch.ones_like(a),))


@pytest.mark.gpu
def test_primals_within_a_dual_level(dev):
    a, b, s = torch.randn(6, 8, device=dev), torch.randn(2, 8, 4, device=dev), torch.tensor([3, 3], device=dev)
    want = gmm(a, b, s)
    with forward_ad.dual_level():
        assert torch.equal(gmm(a, b, s), want)
        dual = forward_ad.make_dual(a, torch.ones_like(a))
        with pytest.raises(RuntimeError, match="forward-mode"):
            gmm(dual, b, s)
        assert torch.equal(gmm(forward_ad.unpack_dual(dual).primal, b, s), want)
        x = torch.randn(6, 5, device=dev)
        assert torch.equal(route(x, 2).experts, torch.topk(x, 2).indices.int())


@pytest.mark.parametrize("need", [(True, True, False), (True, False, False), (False, True, False)])
def test_tangent_of_an_incoming_gradient(monkeypatch, need):
    """Forward over reverse: the loss has a tangent where the product's operands have none."""
    from types import SimpleNamespace

    from triturus_amd import gmm as gmm_module
    from triturus_amd import route as route_module

    for module in (gmm_module, route_module):
        monkeypatch.setattr(module, "refuse_capture", lambda op: None)
    for name in ("_forward", "_weights"):
        monkeypatch.setattr(gmm_module, name, lambda *a: torch.zeros(1))
    monkeypatch.setattr(route_module, "_grad", lambda *a: torch.zeros(1))
    a, b, s, g = torch.randn(6, 8), torch.randn(2, 8, 4), torch.tensor([3, 3]), torch.randn(6, 4)
    ctx = SimpleNamespace(saved_tensors=(a if need[1] else None, b if need[0] else None, s), needs_input_grad=need)
    routes = SimpleNamespace(saved_tensors=(torch.randn(6, 5), torch.rand(6, 2), torch.zeros(6, 2, dtype=torch.int32)), normalize=True)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            gmm_module._Gmm.backward(ctx, forward_ad.make_dual(g, torch.ones_like(g)))
        w = torch.randn(6, 2)
        with pytest.raises(RuntimeError, match="forward-mode"):
            route_module._Route.backward(routes, forward_ad.make_dual(w, torch.ones_like(w)))
        if not (need[0] and need[1]):
            gmm_module._Gmm.backward(ctx, g)
        route_module._Route.backward(routes, w)


@pytest.mark.gpu
@pytest.mark.parametrize("both", [True, False])
def test_forward_over_reverse_on_the_device(dev, both):
    a, b, s = torch.randn(6, 8, device=dev, requires_grad=True), torch.randn(2, 8, 4, device=dev, requires_grad=both), torch.tensor([3, 3], device=dev)
    x, w = torch.randn(6, 5, device=dev, requires_grad=True), torch.randn(6, 4, device=dev)
    with forward_ad.dual_level():
        loss = (gmm(a, b, s) * forward_ad.make_dual(w, torch.ones_like(w))).sum()
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(loss, (a, b) if both else (a,))
        v = torch.randn(6, 2, device=dev)
        loss = (route(x, 2).weights * forward_ad.make_dual(v, torch.ones_like(v))).sum()
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(loss, (x,))
        plain = torch.autograd.grad((gmm(a, b, s) * w).sum(), (a,))[0]
    assert torch.equal(plain, torch.autograd.grad((gmm(a, b, s) * w).sum(), (a,))[0])
