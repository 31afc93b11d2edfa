"""What gmm's autograd function keeps and calls, without a GPU: the products are stood in for by torch's own on the CPU."""

import pytest
import torch

from triturus_amd import gmm as module


def rows_product(a, b, sizes, tile=0):
    c, r = torch.zeros(a.shape[0], b.shape[2]), 0
    for e, n in enumerate(sizes.tolist()):
        c[r:r + n] = a[r:r + n] @ b[e]
        r += n
    return c


def weights_product(a, g, sizes, tile=0):
    d, r = torch.zeros(sizes.shape[0], a.shape[1], g.shape[1]), 0
    for e, n in enumerate(sizes.tolist()):
        d[e] = a[r:r + n].T @ g[r:r + n]
        r += n
    return d


@pytest.fixture
def calls(monkeypatch):
    seen = []

    def spy(name, fn):
        def call(*args, **kw):
            seen.append(name)
            return fn(*args, **kw)

        monkeypatch.setattr(module, name, call)

    spy("_forward", rows_product)
    spy("_weights", weights_product)
    spy("gmm_grad", lambda g, a, b, s: (rows_product(g, b.transpose(1, 2), s), weights_product(a, g, s)))
    monkeypatch.setattr(module, "refuse_capture", lambda op: None)
    return seen


def operands(a_grad, b_grad):
    a, b = torch.randn(7, 5, requires_grad=a_grad), torch.randn(3, 5, 4, requires_grad=b_grad)
    return a, b, torch.tensor([3, 0, 3])


def test_both_gradients_are_one_call(calls):
    a, b, s = operands(True, True)
    c = module._Gmm.apply(a, b, s)
    g = torch.randn_like(c)
    del calls[:]
    c.backward(g)
    assert calls == ["gmm_grad"]
    assert torch.equal(a.grad, rows_product(g, b.detach().transpose(1, 2), s)) and torch.equal(b.grad, weights_product(a.detach(), g, s))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("K,N,dtype", [(257, 130, torch.float16), (64, 131, torch.bfloat16), (40, 56, torch.float32)])
def test_backward_is_gmm_grad(dev, K, N, dtype, layout):
    sizes, T = torch.tensor([300, 0, 400, 3], dtype=torch.int32, device=dev), 710
    a = torch.randn(T, K, device=dev).to(dtype).requires_grad_()
    b = (torch.randn(4, K, N, device=dev) if layout == "kn" else torch.randn(4, N, K, device=dev).transpose(1, 2)).to(dtype).requires_grad_()
    g = torch.randn(T, N, device=dev).to(dtype)
    module.gmm(a, b, sizes).backward(g)
    da, db = module.gmm_grad(g, a.detach(), b.detach(), sizes)
    assert torch.equal(a.grad, da) and torch.equal(b.grad, db)


@pytest.mark.parametrize("a_grad", [True, False])
def test_one_gradient_keeps_one_operand(calls, a_grad):
    """The other operand is neither kept alive nor guarded against changes in place."""
    a, b, s = operands(a_grad, not a_grad)
    c = module._Gmm.apply(a, b, s)
    kept = c.grad_fn.saved_tensors
    assert kept[0] is None if a_grad else kept[1] is None
    g = torch.randn_like(c)
    want = rows_product(g, b.transpose(1, 2), s) if a_grad else weights_product(a, g, s)
    del calls[:]
    with torch.no_grad():
        (a if a_grad else b).mul_(2)  # the operand whose own values its gradient does not need
    c.backward(g)
    assert torch.equal(a.grad if a_grad else b.grad, want)
    assert calls == ["_forward" if a_grad else "_weights"]
