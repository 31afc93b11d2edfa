"""gmm and gmm_grad against the definition in 64 bits.

Tolerance of one value: operands are exact in 64 bits; products of 16-bit values are exact in fp32, fp32
products and every addition round by at most 2^-23 of the running sum of magnitudes (truncation counted), so the
sum is off by at most (terms + 1) 2^-23 sum |x||y|, and the result's own rounding by eps / 2 of its value (and half
the smallest subnormal step of the type).
"""

import math

import pytest
import torch

from triturus_amd.gmm import gmm, gmm_grad

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def product64(a, b, sizes):
    c = torch.zeros(a.shape[0], b.shape[2], dtype=torch.float64, device=a.device)
    r = 0
    for e, n in enumerate(sizes):
        c[r:r + n] = a[r:r + n].double() @ b[e].double()
        r += n
    return c


def weights64(a, g, sizes):
    d, r = [], 0
    for n in sizes:
        d.append(a[r:r + n].double().T @ g[r:r + n].double())
        r += n
    return torch.stack(d)


def close(got, want, magnitude, terms):
    info = torch.finfo(got.dtype)
    bound = (info.eps / 2) * want.abs() + (terms + 1) * 2.0 ** -23 * magnitude + info.smallest_normal * info.eps / 2
    bad = ~((got.double() - want).abs() <= bound * (1 + 2 ** -8))  # the rounding counts the rounded value's binade
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {float((got.double() - want).abs()[bad].max())}"


def operands(dev, T, E, K, N, dtype, layout="kn"):
    a = torch.randn(T, K, device=dev).to(dtype)
    b = (torch.randn(E, K, N, device=dev) if layout == "kn" else torch.randn(E, N, K, device=dev)).to(dtype)
    return a, (b if layout == "kn" else b.transpose(1, 2)), torch.randn(T, N, device=dev).to(dtype)


def check(a, b, g, sizes, wide=False):
    dev = a.device
    s = torch.tensor(sizes, dtype=torch.int64 if wide else torch.int32, device=dev)
    c = gmm(a, b, s)
    assert c.shape == g.shape and c.dtype == a.dtype and c.is_contiguous()
    close(c, product64(a, b, sizes), product64(a.abs(), b.abs(), sizes), a.shape[1])
    da, db = gmm_grad(g, a, b, s)
    assert da.shape == a.shape and db.shape == b.shape and da.dtype == db.dtype == a.dtype
    bt = b.transpose(1, 2)
    close(da, product64(g, bt, sizes), product64(g.abs(), bt.abs(), sizes), b.shape[2])
    close(db, weights64(a, g, sizes), weights64(a.abs(), g.abs(), sizes), max([1] + sizes))
    return c, da, db


SHAPES = [  # sizes, K, N, rows behind the last group
    ([1], 1, 1, 0), ([0], 5, 3, 1), ([1, 0, 1], 8, 8, 0), ([3, 0, 5, 1], 64, 128, 2), ([0, 0, 130], 72, 136, 0),
    ([127, 128, 129, 1], 128, 128, 7), ([257], 200, 264, 0), ([33, 0, 64, 65, 31, 2], 129, 77, 11), ([300, 5], 65, 1, 3),
    ([5, 300], 1, 65, 0), ([16] * 70, 96, 40, 5), ([1] * 130 + [0] * 10 + [40], 64, 64, 0), ([512, 0, 512], 256, 512, 0),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_products_and_gradients(dev, shape, layout, dtype):
    sizes, K, N, tail = SHAPES[shape]
    check(*operands(dev, sum(sizes) + tail, len(sizes), K, N, dtype, layout), sizes, wide=shape % 2 == 1)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,E", [(2, 64), (40, 3), (130, 2), (700, 4), (2500, 5)])
def test_sizes_over_the_tiles(dev, T, E, dtype):
    cut = torch.sort(torch.randint(0, T + 1, (E - 1,)))[0].tolist()
    sizes = [y - x for x, y in zip([0] + cut, cut + [T])]
    for K, N in ((64, 256), (264, 520), (515, 300)):
        check(*operands(dev, T, E, K, N, dtype), sizes)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_views_are_read_in_place(dev, dtype):
    sizes, K, N = [20, 0, 50], 48, 72
    a, b, g = operands(dev, 70, 3, K, N, dtype)
    for off in (0, 1, 8):  # offsets and row lengths that leave and keep 16-byte boundaries
        wide_a, wide_b, wide_g = (torch.full((*t.shape[:-1], t.shape[-1] + 16), math.nan, device=dev, dtype=dtype) for t in (a, b, g))
        va, vb, vg = (w[..., off:off + t.shape[-1]].copy_(t) for w, t in ((wide_a, a), (wide_b, b), (wide_g, g)))
        check(va, vb, vg, sizes)
    check(a[:, ::2], b[:, ::2, ::3], g[:, ::3], sizes)  # no unit stride: copied
    check(a[:1].expand(70, K), b[:1].expand(3, K, N), g[:1].expand(70, N), sizes)
    s = torch.tensor([20, 9, 0, 9, 50], dtype=torch.int32, device=dev)[::2]
    assert torch.equal(gmm(a, b, s), gmm(a, b, s.clone()))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_neighbours_do_not_leak(dev, dtype):
    """NaN and infinity in other groups, in the rows behind the last group and in other matrices stay there."""
    sizes, K, N = [37, 0, 21, 64], 40, 56
    a, b, g = operands(dev, 130, 4, K, N, dtype)
    clean = check(a, b, g, sizes)
    a[37:58], g[37:58], b[1] = math.nan, math.inf, math.nan
    a[122:], g[122:] = math.inf, math.nan
    s = torch.tensor(sizes, device=dev)
    c, (da, db) = gmm(a, b, s), gmm_grad(g, a, b, s)
    keep = torch.ones(130, dtype=torch.bool, device=dev)
    keep[37:58] = False
    assert torch.equal(c[keep], clean[0][keep]) and torch.equal(da[keep], clean[1][keep])
    assert c[37:58].isnan().all() and not c[122:].any() and not da[122:].any()
    assert torch.equal(db[[0, 1, 3]], clean[2][[0, 1, 3]]) and db[2].isnan().all()


@pytest.mark.parametrize("sizes", [[5, -3, 9, 4], [10, 100, 7, 3], [1 << 30, 1 << 30, 1 << 30, 1 << 30], [-1, -1, -1, -1]])
def test_sizes_that_do_not_fit_are_clamped(dev, sizes):
    T, K, N = 40, 24, 32
    a, b, g = operands(dev, T, 4, K, N, torch.float32)
    fit, left = [], T
    for n in sizes:
        fit.append(min(max(n, 0), left))
        left -= fit[-1]
    for dtype in (torch.int32, torch.int64):
        s = torch.tensor(sizes, dtype=dtype, device=dev)
        want = torch.tensor(fit, dtype=dtype, device=dev)
        assert torch.equal(gmm(a, b, s), gmm(a, b, want))
        for x, y in zip(gmm_grad(g, a, b, s), gmm_grad(g, a, b, want)):
            assert torch.equal(x, y)


def test_empty_operands(dev):
    s = torch.tensor([0, 0], device=dev)
    a, b = torch.empty(0, 8, device=dev), torch.randn(2, 8, 4, device=dev)
    assert gmm(a, b, s).shape == (0, 4)
    da, db = gmm_grad(torch.empty(0, 4, device=dev), a, b, s)
    assert da.shape == (0, 8) and not db.any() and db.shape == b.shape
    s = torch.tensor([3, 0], device=dev)
    assert not gmm(torch.empty(5, 0, device=dev), torch.empty(2, 0, 4, device=dev), s).any()
    assert gmm(torch.randn(5, 8, device=dev), torch.empty(2, 8, 0, device=dev), s).shape == (5, 0)
    da, db = gmm_grad(torch.empty(5, 0, device=dev), torch.randn(5, 8, device=dev), torch.empty(2, 8, 0, device=dev), s)
    assert da.shape == (5, 8) and not da.any() and db.shape == (2, 8, 0)


def test_autograd_matches_differences(dev):
    """The gradient of sum(g c) is linear in each operand: c(a + h) - c(a) along a direction, in 64 bits, is exact."""
    sizes = torch.tensor([7, 0, 12], dtype=torch.int32, device=dev)
    a, b, g = operands(dev, 21, 3, 10, 14, torch.float32)
    a.requires_grad_(), b.requires_grad_()
    (gmm(a, b, sizes) * g).sum().backward()
    da, db = torch.randn_like(a), torch.randn_like(b)
    value = lambda x, y: (product64(x, y, [7, 0, 12]) * g.double()).sum()  # noqa: E731
    with torch.no_grad():
        up = value(a.double() + da.double(), b) - value(a, b)
        along = (a.grad.double() * da).sum()
        scale = (product64(g.abs(), b.abs().transpose(1, 2), [7, 0, 12]) * da.abs()).sum()
        assert abs(up - along) <= 16 * 2.0 ** -23 * scale
        up = value(a, b.double() + db.double()) - value(a, b)
        along = (b.grad.double() * db).sum()
        scale = (weights64(a.abs(), g.abs(), [7, 0, 12]) * db.abs()).sum()
        assert abs(up - along) <= 22 * 2.0 ** -23 * scale
    # one operand alone, a product that is summed (an expanded gradient), a shared matrix
    x = a.detach().clone().requires_grad_()
    gmm(x, b.detach(), sizes).sum().backward()
    assert torch.equal(x.grad, gmm_grad(torch.ones_like(g), x.detach(), b.detach(), sizes)[0])
    w = b.detach()[:1].clone().requires_grad_()
    (gmm(a.detach(), w.expand(3, -1, -1), sizes) * g).sum().backward()
    each = gmm_grad(g, a.detach(), w.detach().expand(3, -1, -1), sizes)[1]
    assert torch.equal(w.grad, each.sum(0, keepdim=True))


def test_graph_and_streams(dev):
    sizes = [100, 0, 60, 40]
    a, b, g = operands(dev, 210, 4, 96, 136, torch.bfloat16)
    s = torch.tensor(sizes, device=dev)
    want = (gmm(a, b, s), *gmm_grad(g, a, b, s))
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = (gmm(a, b, s), *gmm_grad(g, a, b, s))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, other))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = (gmm(a, b, s), *gmm_grad(g, a, b, s))
    for turn in ([50, 50, 50, 50], [0, 200, 10, 0], sizes):  # sizes change between replays
        s.copy_(torch.tensor(turn))
        eager = (gmm(a, b, s), *gmm_grad(g, a, b, s))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, eager))
    with pytest.raises(RuntimeError, match="capture"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            gmm(a.clone().requires_grad_(), b, s)
    torch.cuda.synchronize()
    assert torch.equal(gmm(a, b, s), want[0])


def test_refusals(dev):
    a, b, g = operands(dev, 6, 2, 8, 4, torch.float32)
    s = torch.tensor([3, 3], device=dev)
    for bad in ((a[0], b, s), (a, b[0], s), (a, b, s[None]), (a[:, :7], b, s), (a, b, s[:1]), (a.half(), b, s), (a, b, s.float()),
                (a, b, s.cpu()), (a, b[:0], s[:0])):
        with pytest.raises(AssertionError):
            gmm(*bad)
    with pytest.raises(NotImplementedError):
        gmm(a.double(), b.double(), s)
    for bad in (g[:, :3], g.half(), g.cpu()):
        with pytest.raises(AssertionError):
            gmm_grad(bad, a, b, s)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tile", range(1, 6))
def test_every_tile(dev, tile, dtype):
    """Each tile on sizes that it would not be chosen for, aligned and not."""
    from triturus_amd.gmm import _forward, _weights

    for sizes, K, N, tail in (([3, 0, 5, 1], 64, 128, 2), ([33, 0, 64, 65, 31, 2], 129, 77, 11), ([300, 5], 648, 264, 3), ([1] * 70, 40, 8, 0), ([2, 257], 1031, 66, 0)):
        for layout in ("kn", "nk"):
            a, b, g = operands(dev, sum(sizes) + tail, len(sizes), K, N, dtype, layout)
            s = torch.tensor(sizes, device=dev)
            close(_forward(a, b, s, tile), product64(a, b, sizes), product64(a.abs(), b.abs(), sizes), K)
            close(_weights(a, g, s, tile), weights64(a, g, sizes), weights64(a.abs(), g.abs(), sizes), max(sizes))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("N", [40, 500, 2000, 6000])
def test_few_rows_over_many_columns(dev, N, dtype):
    """One or two rows under the widths at which a tile of few rows changes its columns or wavefronts."""
    for K in (8, 264, 2056):
        for layout in ("kn", "nk"):
            check(*operands(dev, 3, 2, K, N, dtype, layout), [2, 1])


def test_many_groups_and_saturating_sizes(dev):
    """More groups than a wavefront has lanes, with sums of sizes beyond 32 bits."""
    E, K, N = 200, 16, 24
    a, b, g = operands(dev, 500, E, K, N, torch.float32)
    sizes = [(7 * e) % 6 for e in range(E)]
    sizes[-1] += 500 - sum(sizes) if sum(sizes) < 500 else 0
    while sum(sizes) > 500:
        sizes[max(range(E), key=lambda e: sizes[e])] -= 1
    check(a, b, g, sizes)
    big = [3] * 150 + [2 ** 31 - 1] * 50
    s = torch.tensor(big, dtype=torch.int32, device=dev)
    fit = torch.tensor([3] * 150 + [50] + [0] * 49, dtype=torch.int32, device=dev)
    assert torch.equal(gmm(a, b, s), gmm(a, b, fit))
    assert torch.equal(gmm_grad(g, a, b, s.long())[1], gmm_grad(g, a, b, fit)[1])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tile", range(1, 6))
def test_neighbours_do_not_leak_from_any_tile(dev, tile, dtype):
    """NaN next to a group's rows, in the next matrix and behind the last group: contractions and tiles that end inside a step
    read none of it, with operands on and off 16-byte boundaries."""
    from triturus_amd.gmm import _forward, _weights

    for sizes, K, N in (([37, 0, 21, 64], 40, 56), ([37, 0, 21, 64], 41, 55), ([130, 1, 70, 3], 264, 328), ([300, 7, 10, 290], 333, 270)):
        T = sum(sizes) + 9
        for layout in ("kn", "nk"):
            a, b, g = operands(dev, T, 4, K, N, dtype, layout)
            s = torch.tensor(sizes, device=dev)
            clean, grad = _forward(a, b, s, tile), _weights(a, g, s, tile)
            lo, hi = sizes[0], sizes[0] + sizes[1] + sizes[2]
            keep = torch.ones(T, dtype=torch.bool, device=dev)
            if sizes[1] == 0:
                a[lo:hi], g[lo:hi], b[2] = math.nan, math.nan, math.nan
                keep[lo:hi] = False
            b[1] = math.nan if sizes[1] == 0 else b[1]
            a[T - 9:], g[T - 9:] = math.nan, math.inf
            c, d = _forward(a, b, s, tile), _weights(a, g, s, tile)
            assert torch.equal(c[keep], clean[keep]) and not c[T - 9:].any()
            live = [0, 1, 3] if sizes[1] == 0 else [0, 1, 2, 3]
            assert torch.equal(d[live], grad[live])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_far_apart(dev, dtype):
    """Rows of long sequences' last tokens, and matrices' rows, further apart than a tile's 31-bit offsets reach."""
    far, K, N = (1 << 23) // torch.finfo(dtype).bits * 8 + 8, 40, 24  # values; one more chunk than the limit
    a, b, g = operands(dev, 3, 2, K, N, dtype)
    wide = [torch.empty(t.shape[0] if t.dim() == 2 else 2 * t.shape[1], far, dtype=dtype, device=dev) for t in (a, b, g)]
    av, gv = wide[0][:, :K].copy_(a), wide[2][:, :N].copy_(g)
    bv = wide[1].view(2, K, far)[:, :, :N].copy_(b)
    for rows in (3, 1):
        sizes = [rows - 1, 1]
        for got, want in zip(check(av[:rows], bv, gv[:rows], sizes), check(a[:rows], b, g[:rows], sizes)):
            assert torch.equal(got, want)


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("sizes,N", [([300, 2, 500], 1500), ([300, 0, 1500, 700], 2000), ([900, 1100, 600, 700], 4000)])
def test_rounds_of_the_largest_tile(dev, sizes, N, layout):
    """Last rounds in quarters, in halves and behind whole ones, under contractions that end at every step of the loop."""
    from triturus_amd.gmm import _forward, _weights

    for K in (8, 64, 96, 128, 136, 256, 328):
        a, b, g = operands(dev, sum(sizes) + 5, len(sizes), K, N, torch.bfloat16, layout)
        s = torch.tensor(sizes, device=dev)
        close(_forward(a, b, s, 5), product64(a, b, sizes), product64(a.abs(), b.abs(), sizes), K)
    close(_weights(a, g, s, 5), weights64(a, g, sizes), weights64(a.abs(), g.abs(), sizes), max(sizes))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("sizes,K,N", [([5000], 96, 200), ([4500, 0, 31, 2000], 130, 257), ([3000, 3000], 129, 64), ([0, 7000], 8, 8), ([9001], 1, 1), ([40] * 66 + [20000] + [700] * 3, 48, 40),
                                       ([1000] * 66 + [20000] + [2500] * 3, 48, 40)])
def test_rows_cut_into_pieces(dev, sizes, K, N, dtype):
    """The matrices' gradient of few and of many long groups, with and without the workspace that the cut takes, and replayed."""
    from triturus_amd import _lib
    from triturus_amd.gmm import _weights

    a, b, g = operands(dev, sum(sizes) + 3, len(sizes), K, N, dtype)
    a[-3:], g[-3:] = math.nan, math.inf
    s = torch.tensor(sizes, device=dev)
    lib, code = _lib.load(), _lib.DTYPE_CODES[dtype]
    T, E = a.shape[0], len(sizes)
    want, size = weights64(a, g, sizes), weights64(a.abs(), g.abs(), sizes)
    d = _weights(a, g, s)
    wanted = lib.trt_gmm_weights_workspace_bytes(a.data_ptr(), g.data_ptr(), T, E, K, N, K, N, code, 0)
    assert wanted >= 65536 * (E + 1) or T < 400 * E  # short groups on average are not cut
    close(d, want, size, max(sizes))
    assert torch.equal(gmm_grad(g, a, b, s)[1], d)
    plain = torch.full_like(d, math.nan)
    assert lib.trt_gmm_weights(a.data_ptr(), g.data_ptr(), s.data_ptr(), plain.data_ptr(), T, E, K, N, K, N, code, 1, 0, None, 0,
                               _lib.raw_stream(dev)) == 0
    close(plain, want, size, max(sizes))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _weights(a, g, s)
    for _ in range(3):
        captured.zero_()
        eager = _weights(a, g, s)
        graph.replay()
        assert torch.equal(captured, d) and torch.equal(eager, d)


@pytest.mark.parametrize("layout", ["kn", "nk"])
@pytest.mark.parametrize("K,N", [(257, 130), (256, 131), (259, 128)])
def test_gradients_with_and_without_copies(dev, K, N, layout):
    """Operands off the boundaries, all or one of them: copied once for both products, or read as they lie without a workspace."""
    from triturus_amd import _lib

    sizes, dtype = [500, 0, 700, 3], torch.float16
    a, b, g = operands(dev, sum(sizes) + 2, len(sizes), K, N, dtype, layout)
    s, bt = torch.tensor(sizes, device=dev, dtype=torch.int32), b.transpose(1, 2)
    lib, code, T, E = _lib.load(), _lib.DTYPE_CODES[dtype], a.shape[0], len(sizes)
    args = g.data_ptr(), a.data_ptr(), b.data_ptr()
    assert lib.trt_gmm_grad_workspace_bytes(*args, T, E, K, N, N, K, _lib.strides3(b), code) > 0
    da, db = torch.full_like(a, math.nan), torch.full((E, K, N), math.nan, dtype=dtype, device=dev)
    assert lib.trt_gmm_grad(*args, s.data_ptr(), da.data_ptr(), db.data_ptr(), T, E, K, N, N, K, _lib.strides3(b), code, 0, None, 0,
                            _lib.raw_stream(dev)) == 0
    for got in ((da, db), gmm_grad(g, a, b, s)):
        close(got[0], product64(g, bt, sizes), product64(g.abs(), bt.abs(), sizes), N)
        close(got[1], weights64(a, g, sizes), weights64(a.abs(), g.abs(), sizes), max(sizes))
