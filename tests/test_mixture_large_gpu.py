"""Operands and results of the mixture layer's operators past 2^31 elements and 4 GiB: the far end against the same rows alone."""

import pytest
import torch

from triturus_amd.gmm import gmm, gmm_grad
from triturus_amd.mx4 import MX4, mm_mx4, mx4_dequantize, mx4_quantize
from triturus_amd.route import Routes, route, route_grad

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _free():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("K,N", [(96, 72), (97, 71)])
def test_gmm_operands_far_apart(dev, K, N):
    """Rows nearly 8 MiB apart and matrices more than 4 GiB apart, on and off the boundaries, are read in place."""
    T, far, group = 600, (1 << 22) - 8, (1 << 31) + 8
    a, b, g = (torch.randn(*s, device=dev).bfloat16() for s in ((T, K), (3, K, N), (T, N)))
    rows = torch.empty(2, T, far, dtype=torch.bfloat16, device=dev)
    av, gv = rows[0, :, :K].copy_(a), rows[1, :, :N].copy_(g)
    bv = torch.empty(2 * group + K * N, dtype=torch.bfloat16, device=dev).as_strided((3, K, N), (group, N, 1)).copy_(b)
    s = torch.tensor([200, 1, 390], device=dev)
    assert torch.equal(gmm(av, bv, s), gmm(a, b, s))
    for x, y in zip(gmm_grad(gv, av, bv, s), gmm_grad(g, a, b, s)):
        assert torch.equal(x, y)


def test_gmm_results_beyond_4_gib(dev):
    T, K, N, half = 70000, 16, 40000, 35000
    a, b = torch.randn(T, K, device=dev).bfloat16(), torch.randn(2, K, N, device=dev).bfloat16()
    s, one = torch.tensor([half, half - 10], device=dev), torch.tensor([64], device=dev)
    c = gmm(a, b, s)
    assert c.numel() > 1 << 31
    for r, e in ((0, 0), (half - 64, 0), (half, 1), (T - 74, 1)):
        x, w = a[r:r + 64].double(), b[e].double()
        # K products exact in fp32, sums within (K + 1) 2^-23 of the magnitudes, one rounding to bf16
        bound = (K + 1) * 2.0 ** -23 * (x.abs() @ w.abs()) + 2.0 ** -8 * (1 + 2 ** -8) * (x @ w).abs()
        assert ((c[r:r + 64].double() - x @ w).abs() <= bound).all()
    assert not c[T - 10:].any()
    da, db = gmm_grad(c, a, b, s)  # c: any incoming gradient of that size
    for r, e in ((0, 0), (half, 1), (T - 74, 1)):
        x, w = c[r:r + 64].double(), b[e].double().T
        bound = (N + 1) * 2.0 ** -23 * (x.abs() @ w.abs()) + 2.0 ** -8 * (1 + 2 ** -8) * (x @ w).abs()
        assert ((da[r:r + 64].double() - x @ w).abs() <= bound).all()
    assert not da[T - 10:].any()
    for e, rows in ((0, slice(0, half)), (1, slice(half, T - 10))):
        x, y = a[rows].double().T, c[rows, -50:].double()
        bound = (half + 1) * 2.0 ** -23 * (x.abs() @ y.abs()) + 2.0 ** -8 * (1 + 2 ** -8) * (x @ y).abs()
        assert ((db[e, :, -50:].double() - x @ y).abs() <= bound).all()


@pytest.mark.parametrize("tile", range(0, 5))
def test_codes_far_apart(dev, tile):
    """Rows of codes nearly 8 MiB apart, matrices and scales more than 4 GiB apart."""
    T, N, K, E = 600, 200, 160, 2
    a, b = mx4_quantize(torch.randn(T, K, device=dev)), mx4_quantize(torch.randn(E, N, K, device=dev))
    far, group = (1 << 23) - 16, (1 << 32) + 16

    def apart(t, stride):
        room = torch.zeros(stride * (t.shape[0] - 1) + t[0].numel(), dtype=torch.uint8, device=dev)
        return room.as_strided(t.shape, (stride, *t.stride()[1:])).copy_(t)

    av = MX4(apart(a.codes, far), apart(a.scales, far), K)
    bv = MX4(apart(b.codes, group), apart(b.scales, group), K)
    s = torch.tensor([300, 295], device=dev)
    assert torch.equal(mm_mx4(av, bv, s, _tile=tile), mm_mx4(a, b, s, _tile=tile))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
def test_quantisation_in_several_launches(dev, dtype):
    """More than 2^30 lanes' work: rows of windows of one line, the ones around the second launch's first against themselves alone."""
    K, first = 256, 1 << 25  # rows of the first launch
    rows = first + 1000
    line = torch.randn(rows + K, device=dev).to(dtype)
    line[first - 7] = 3e38 if dtype == torch.float32 else 1e30
    x = line.as_strided((rows, K), (1, 1))
    q = mx4_quantize(x)
    for r in (0, first - 500, rows - 500):
        part = mx4_quantize(x[r:r + 500].contiguous())
        assert torch.equal(q.codes[r:r + 500], part.codes) and torch.equal(q.scales[r:r + 500], part.scales)
    y = mx4_dequantize(q, dtype=torch.bfloat16)
    for r in (0, first - 500, rows - 500):
        part = MX4(q.codes[r:r + 500].clone(), q.scales[r:r + 500].clone(), K)
        assert torch.equal(y[r:r + 500], mx4_dequantize(part, dtype=torch.bfloat16))


def test_route_beyond_4_gib(dev):
    T, E, k = (1 << 22) + 77, 1024, 2
    x = torch.randn(T, E, device=dev, dtype=torch.bfloat16)
    r = route(x, k, normalize=False)
    assert int(r.sizes.sum()) == T * k
    last = slice(T - 3000, T)
    part = route(x[last].clone(), k, normalize=False)
    assert torch.equal(r.experts[last], part.experts) and torch.equal(r.weights[last], part.weights)
    assert torch.equal(torch.bincount(r.experts.flatten().long(), minlength=E).int(), r.sizes)
    at = r.slots.flatten().long()
    assert torch.equal(r.rows[at], torch.arange(T, device=dev, dtype=torch.int32).repeat_interleave(k))
    starts = r.sizes.long().cumsum(0) - r.sizes
    place = at - starts[r.experts.flatten().long()]
    assert (place >= 0).all() and (place < r.sizes[r.experts.flatten().long()]).all() and torch.equal(at.sort()[0], torch.arange(T * k, device=dev))
    g = torch.randn(T, k, device=dev)
    d = route_grad(g, x, r, normalize=False)
    alone = Routes(r.weights[last].clone(), r.experts[last].clone(), r.rows, r.slots, r.sizes)
    assert torch.equal(d[last], route_grad(g[last].clone(), x[last].clone(), alone, normalize=False))
