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
