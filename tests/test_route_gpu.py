"""route and route_grad against the definition in 64 bits on the CPU, and a mixture layer put together from all its operators.

Whole numbers are equal.  A weight e^(x - m) / sum is off by: x - m rounds once (2^-24 of it, times the exponential's
slope), the exponential is within 2 units in the last place, the sum of n terms within n 2^-24, the quotient 2^-24 --
(|x - m| + n + 6) 2^-24 of the weight in all; the smallest exponentials flush below 2^-126.
"""

import math

import pytest
import torch

from triturus_amd.gmm import gmm, gmm_grad
from triturus_amd.mx4 import mm_mx4, mx4_dequantize, mx4_quantize
from triturus_amd.route import Routes, route, route_grad

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def route64(x, k, normalize):
    x = x.double().cpu()
    T, E = x.shape
    rank = x.nan_to_num(math.inf, posinf=1e300)  # NaN above all; no +inf beside it in these tests
    top, at = torch.sort(rank, dim=1, descending=True, stable=True)
    at = at[:, :k]
    value = x.gather(1, at)
    live = value != -math.inf
    m = value[:, :1]
    e = torch.where(live, torch.exp(value - m), 0.0)
    total = e.sum(1, keepdim=True) if normalize else torch.where(x != -math.inf, torch.exp(x - m), 0.0).sum(1, keepdim=True)
    weights = torch.where(live, e / total, 0.0)
    experts = torch.where(live, at, -1)
    flat = experts.flatten().tolist()
    order = sorted((i for i, e in enumerate(flat) if e >= 0), key=lambda i: (flat[i], i))
    rows = torch.zeros(T * k, dtype=torch.int32)
    slots = torch.full((T * k,), -1, dtype=torch.int32)
    for place, i in enumerate(order):
        rows[place] = i // k
        slots[i] = place
    sizes = torch.bincount(torch.tensor([e for e in flat if e >= 0], dtype=torch.long), minlength=E).int()
    return Routes(weights, experts.int(), rows, slots.view(T, k), sizes), (value - m).where(live, 0.0).abs()


def check(x, k, normalize):
    r = route(x, k, normalize=normalize)
    want, far = route64(x, k, normalize)
    for name in ("experts", "rows", "slots", "sizes"):
        got = getattr(r, name)
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), getattr(want, name)), name
    w = r.weights.cpu().double()
    assert r.weights.dtype == torch.float32 and torch.equal(w.isnan(), want.weights.isnan())
    bound = (far + x.shape[1] + 6) * 2.0 ** -24 * want.weights + 2.0 ** -126
    assert not ((w - want.weights).abs() > bound).any()
    return r, want


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (3, 5, 5), (64, 64, 2), (65, 60, 4), (63, 128, 8), (200, 130, 7), (300, 16, 16), (130, 257, 3),
                                   (70, 512, 16), (67, 1000, 10), (129, 1024, 1), (4096, 40, 3), (4097, 33, 2), (9000, 72, 6)])
def test_choice_and_order(dev, T, E, k, dtype):
    x = (2 * torch.randn(T, E, device=dev)).to(dtype)
    for normalize in (True, False):
        check(x, k, normalize)


@pytest.mark.parametrize("E,k", [(8, 3), (100, 8), (300, 16)])
def test_ties_masks_and_specials(dev, E, k):
    x = torch.randint(-2, 3, (200, E), device=dev).float()  # many equal values
    x[x == 0] = torch.where(torch.rand(200, E, device=dev)[x == 0] < 0.5, 0.0, -0.0)  # equal too
    check(x, k, True)
    x[torch.rand(200, E, device=dev) < 0.7] = -math.inf  # fewer than k are left now and then
    x[3] = x[150] = -math.inf
    x[5] = -math.inf
    x[5, E - 1] = -3e38
    for normalize in (True, False):
        r, _ = check(x, k, normalize)
        assert (r.experts[3] == -1).all() and not r.weights[3].any() and (r.slots[3] == -1).all()
        assert r.experts[5].tolist() == [E - 1] + [-1] * (k - 1) and r.weights[5, 0] == 1
    x[7, 2], x[7, 4] = math.nan, math.nan
    x[8, 6] = math.nan
    r, _ = check(x, k, True)
    assert r.experts[7, :2].tolist() == [2, 4] and r.weights[8, 0].isnan()
    x = torch.full((70, E), -math.inf, device=dev)
    r, _ = check(x, k, True)
    assert not r.sizes.any() and not r.rows.any()
    x[9, 1] = math.inf
    r = route(x, k)
    assert r.experts[9, 0] == 1 and r.weights[9, 0].isnan() and r.sizes.sum() == 1
    check(1e4 * torch.randn(100, E, device=dev), k, True)  # far apart
    check(3e38 * torch.rand(100, E, device=dev), k, False)


def test_strides(dev):
    wide = torch.randn(100, 90, device=dev)
    for x in (wide[:, 3:43], wide[::2, :40], wide[:, ::2], wide[:1].expand(70, 90), wide.T):
        a, b = route(x, 4), route(x.contiguous(), 4)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
    g = torch.randn(100, 4, device=dev)
    x = wide[:, 3:43]
    r = route(x, 4, normalize=False)
    assert torch.equal(route_grad(g, x, r, normalize=False), route_grad(g, x.contiguous(), r, normalize=False))
    assert torch.equal(route_grad(g[:, :1].expand(100, 4), x, r), route_grad(g[:, :1].expand(100, 4).contiguous(), x, r))


@pytest.mark.parametrize("normalize", [True, False])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (5, 8, 2), (70, 65, 8), (33, 130, 16), (40, 300, 5), (17, 1024, 6), (17, 1001, 6)])
def test_gradient(dev, T, E, k, dtype, normalize):
    x = (2 * torch.randn(T, E, device=dev)).to(dtype)
    x[torch.rand(T, E, device=dev) < 0.2] = -math.inf
    g = torch.randn(T, k, device=dev)
    y = x.clone().requires_grad_()
    r = route(y, k, normalize=normalize)
    (r.weights * g).sum().backward()
    d = route_grad(g, x, route(x, k, normalize=normalize), normalize=normalize)
    assert d.dtype == dtype and torch.equal(d, y.grad)
    want, far = route64(x, k, normalize)
    w, gd = want.weights, g.cpu().double()
    inner = (w * gd).sum(1, keepdim=True)
    at = want.experts.long().clamp(min=0)
    live = want.experts >= 0
    xd = x.cpu().double()
    m = xd.amax(1, keepdim=True)
    p = torch.where(xd != -math.inf, torch.exp(xd - m), 0.0)
    p = torch.where(p.sum(1, keepdim=True) > 0, p / p.sum(1, keepdim=True), 0.0).nan_to_num(0.0)
    full = torch.zeros(T, E, dtype=torch.float64) if normalize else -p * inner
    full.scatter_add_(1, at, torch.where(live, w * (gd - inner) if normalize else w * gd, 0.0))
    # weights as above, the sum over choices and the difference two more roundings of at most |w|(|g| + sum |w g|), and the type's own
    size = torch.zeros(T, E, dtype=torch.float64) if normalize else p * (w * gd).abs().sum(1, keepdim=True)
    size.scatter_add_(1, at, torch.where(live, w * (gd.abs() + (w * gd).abs().sum(1, keepdim=True)), 0.0))
    info = torch.finfo(dtype)
    spread = (xd - m).abs().nan_to_num(0.0, posinf=0.0).amax(1, keepdim=True)
    bound = full.abs() * info.eps / 2 * (1 + 2 ** -8) + 2 * (spread + E + k + 12) * 2.0 ** -24 * size + info.smallest_normal * info.eps / 2 + 2.0 ** -120
    assert not ((d.cpu().double() - full).abs() > bound).any()


def test_gradient_against_differences(dev):
    x, g = torch.randn(30, 20, device=dev), torch.randn(30, 4, device=dev)
    for normalize in (True, False):
        d = route_grad(g, x, route(x, 4, normalize=normalize), normalize=normalize).cpu().double()
        u = torch.randn(30, 20, dtype=torch.float64)
        h = 1e-6  # the choice stays: equal choices are checked
        up, down = (route64(x.cpu().double() + s * h * u, 4, normalize)[0] for s in (1, -1))
        assert torch.equal(up.experts, down.experts)
        slope = ((up.weights - down.weights) * g.cpu().double()).sum() / (2 * h)
        # third derivatives of a softmax are below 1: h^2 |u|^3 |g| / 6 apart, and the gradient's own 1e-6
        assert abs(slope - (d * u).sum()) <= 1e-5 * (1 + (d * u).abs().sum())


def test_empty_and_refusals(dev):
    r = route(torch.empty(0, 8, device=dev), 2)
    assert r.weights.shape == (0, 2) and r.rows.shape == (0,) and not r.sizes.any()
    x = torch.randn(4, 8, device=dev)
    for bad in ((x[0], 1), (x, 0), (x, 9)):
        with pytest.raises(AssertionError):
            route(*bad)
    with pytest.raises(NotImplementedError):
        route(x.double(), 2)
    for E, k in ((1025, 2), (40, 17)):
        with pytest.raises(RuntimeError, match="range"):
            route(torch.randn(3, E, device=dev), k)
    r, g = route(x, 2), torch.randn(4, 2, device=dev)
    for args in ((g[:, :1], x, r), (g.half(), x, r), (g[:3], x, r), (g, x[:3], r), (g.cpu(), x, r)):
        with pytest.raises(AssertionError):
            route_grad(*args)
    # experts that are not this router's take no gradient
    assert not route_grad(g, x, r._replace(experts=torch.full_like(r.experts, 8))).any()


def layer(x, logits, w1, w2, k):
    r = route(logits, k)
    h = gmm(x[r.rows], w1, r.sizes)
    y = gmm(torch.nn.functional.silu(h), w2, r.sizes)
    return (y[r.slots].float() * r.weights[..., None]).sum(1), r


def layer64(x, logits, w1, w2, k):
    r, _ = route64(logits.detach(), k, True)
    x, w1, w2, l = (t.double().cpu() for t in (x, w1, w2, logits))
    live = (r.experts >= 0)
    chosen = l.gather(1, r.experts.long().clamp(min=0)).masked_fill(~live, -math.inf)
    weights = torch.where(live.any(1, keepdim=True), torch.softmax(chosen.masked_fill(~live.any(1, keepdim=True), 0.0), 1), 0.0)
    out = []
    for t in range(x.shape[0]):
        o = torch.zeros(w2.shape[2], dtype=torch.float64)
        for j, e in enumerate(r.experts[t].tolist()):
            if e >= 0:
                o = o + weights[t, j] * (torch.nn.functional.silu(x[t] @ w1[e]) @ w2[e])
        out.append(o)
    return torch.stack(out)


def test_mixture_layer(dev):
    """Router, grouped products and the weighted sum together: values and gradients, padded rows among them, and a captured step."""
    T, E, k, K, H = 50, 6, 2, 24, 40
    x, logits = torch.randn(T, K, device=dev), torch.randn(T, E, device=dev)
    logits[4] = -math.inf  # a padded row
    logits[:, 3] = -math.inf  # an expert that nobody may choose
    w1, w2 = torch.randn(E, K, H, device=dev) / K ** 0.5, torch.randn(E, H, K, device=dev) / H ** 0.5
    ours, exact = [[t.detach().clone().to(d).requires_grad_() for t in (x, logits, w1, w2)] for d in (torch.float32, torch.float64)]
    y, r = layer(*ours, k)
    want = layer64(*exact, k)
    # every value is a sum of at most K H k products of O(1) numbers in fp32: 2^-24 times some hundred
    assert (y.detach().cpu().double() - want.detach()).abs().max() < 1e-4
    assert not y[4].any() and r.sizes[3] == 0 and r.sizes.sum() == (T - 1) * k
    g = torch.randn_like(y)
    (y * g).sum().backward()
    (want * g.cpu().double()).sum().backward()
    for a, b in zip(ours, exact):
        scale = b.grad.abs().max()
        assert ((a.grad.double() - b.grad).abs().max() / scale) < 1e-4
    assert not ours[2].grad[3].any() and not ours[0].grad[4].any()
    # captured: forward and backward by the functions that take no part in autograd
    x, logits, w1, w2 = (t.detach() for t in ours)

    def step():
        r = route(logits, k)
        xs = x[r.rows]
        h = gmm(xs, w1, r.sizes)
        dh, dw = gmm_grad(torch.ones_like(h), xs, w1, r.sizes)
        dl = route_grad(torch.ones_like(r.weights), logits, r)
        return h, dh, dw, dl, *r

    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        x.normal_(), logits.normal_()
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, eager))
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            route(logits.clone().requires_grad_(), k)
    torch.cuda.synchronize()


def test_mixture_layer_in_4_bits(dev):
    """Router and 4-bit products: the same as fp32 products of the 4-bit values, up to the fp32 sums."""
    T, E, k, K, N = 40, 5, 2, 96, 72
    x, r = torch.randn(T, K, device=dev), route(torch.randn(T, E, device=dev), 2)
    w = mx4_quantize(torch.randn(E, N, K, device=dev))
    rows = x[r.rows]
    got = mm_mx4(rows, w, r.sizes)
    xv, wv = mx4_dequantize(mx4_quantize(rows)), mx4_dequantize(w).transpose(1, 2)
    want = gmm(xv, wv, r.sizes)
    bound = 2 * (K + 2) * 2.0 ** -23 * gmm(xv.abs(), wv.abs().contiguous(), r.sizes)
    assert ((got - want).abs() <= bound).all()


def test_streams(dev):
    x = torch.randn(5000, 64, device=dev)
    want = route(x, 4)
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(route(x, 4))
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for o in outs for p, q in zip(o, want))


def test_results_changed_in_place(dev):
    """A result changed in place spoils nothing that autograd saved of the others."""
    logits = torch.randn(70, 9, device=dev)
    logits[3] = -math.inf
    x, g = torch.randn(70, 8, device=dev, requires_grad=True), torch.randn(70, 2, device=dev)
    want = route_grad(g, logits, route(logits, 2))
    leaf = logits.clone().requires_grad_()
    r = route(leaf, 2)
    y = x[r.rows]
    r.slots.clamp_(min=0), r.sizes.add_(1)
    (r.weights * g).sum().backward()
    assert torch.equal(leaf.grad, want)
    r = route(logits, 2)
    y = x[r.rows]
    r.weights.mul_(2.5), r.experts.clamp_(min=0)
    y.sum().backward()
    assert torch.equal(x.grad.sum(1), 8.0 * torch.bincount(r.rows.long(), minlength=70))
