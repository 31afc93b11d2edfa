"""The microscaled 4-bit format: codes and scales bit for bit, products against 64 bits.

Products of two 4-bit values under their scales are exact, so a product's value is off by the fp32 sums, at most
(terms + 1) 2^-23 sum |x||y| (truncation counted), and by half a step of its own type.
"""

import math

import pytest
import torch

from triturus_amd.mx4 import MX4, mm_mx4, mx4_dequantize, mx4_quantize

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def quantize64(x):
    """Codes (one a byte) and scales by the definition, in 64 bits on the CPU."""
    K = x.shape[-1]
    x = torch.nn.functional.pad(x.double().cpu(), (0, -K % 32)).unflatten(-1, (-1, 32))
    top = x.abs().amax(-1)
    special = ~torch.isfinite(top)
    e = torch.where(special | (top == 0), -127, (torch.frexp(top)[1] - 3).clamp(-127, 127))
    v = x * torch.pow(torch.tensor(2.0, dtype=torch.float64), -e.double()).unsqueeze(-1)
    table = torch.tensor(VALUES, dtype=torch.float64)
    distance = (v.abs().unsqueeze(-1) - table).abs()
    nearest = distance.amin(-1, keepdim=True)
    both = distance == nearest  # one code, or two neighbours, of which the even one is taken
    even = torch.arange(8) % 2 == 0
    code = torch.where(both.sum(-1) > 1, (both & even).to(torch.uint8).argmax(-1), both.to(torch.uint8).argmax(-1))
    code = code + 8 * torch.signbit(x)
    code[special] = 0
    return code.to(torch.uint8), torch.where(special, 255, e + 127).to(torch.uint8)


def unpack(q):
    c = q.codes.cpu()
    return torch.stack((c & 15, c >> 4), -1).flatten(-2).unflatten(-1, (-1, 32)), q.scales.cpu()


def values64(q):
    code, scale = unpack(q)
    v = torch.tensor(VALUES, dtype=torch.float64)[(code & 7).long()] * torch.where(code >= 8, -1.0, 1.0)
    v = v * torch.pow(torch.tensor(2.0, dtype=torch.float64), scale.double() - 127).unsqueeze(-1)
    v[scale == 255] = math.nan
    return v.flatten(-2)[..., :q.length]


def same_codes(q, x):
    code, scale = quantize64(x)
    got, got_scale = unpack(q)
    assert torch.equal(got_scale, scale)
    wrong = got != code
    assert not wrong.any(), f"{int(wrong.sum())} codes differ, first {got[wrong][0]} for {code[wrong][0]}"


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 1), (3, 31), (2, 32), (5, 33), (1, 4096), (7, 1000), (65, 72), (2, 3, 40), (129, 256), (50,)], ids=str)
def test_quantize_and_back(dev, shape, dtype):
    x = (torch.randn(*shape, device=dev) * torch.exp(3 * torch.randn(*shape[:-1], 1, device=dev))).to(dtype)
    q = mx4_quantize(x)
    blocks = -(-shape[-1] // 32)
    assert q.codes.shape == (*shape[:-1], 16 * blocks) and q.scales.shape == (*shape[:-1], blocks) and q.length == shape[-1]
    same_codes(q, x)
    for out in TYPES:
        y = mx4_dequantize(q, dtype=out)
        assert y.shape == x.shape and y.dtype == out
        assert torch.equal(y.cpu(), values64(q).to(out))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_every_tie_and_binade(dev, dtype):
    """Each value, each midpoint and their neighbours in the type, of both signs, under scales over the type's whole range."""
    info = torch.finfo(dtype)
    mids = [(p + q) / 2 for p, q in zip(VALUES, VALUES[1:])]
    base = torch.tensor(sorted(VALUES + mids + [5.5, 7.0, 7.5]), dtype=torch.float64)
    rows = []
    lowest = int(math.log2(info.smallest_normal * info.eps))
    for e in range(lowest - 2, int(math.log2(info.max)) - 1):
        for top in (4.0, 6.0, 7.5):
            v = base[base <= top] * 2.0 ** e
            v = v.to(dtype)
            near = [v, torch.nextafter(v, torch.full_like(v, math.inf)), torch.nextafter(v, torch.zeros_like(v))] if dtype != torch.bfloat16 else [
                v, (v.view(torch.int16) + 1).view(dtype), (v.view(torch.int16) - 1).clamp(min=0).view(dtype)]
            for n in near:
                n = n[n.double() <= top * 2.0 ** e] if dtype == torch.float32 else n
                row = torch.zeros(32, dtype=dtype)
                row[:min(n.numel(), 30)] = n[:30]
                row[30], row[31] = top * 2.0 ** e, 0.0
                rows += [row, -row]
    x = torch.stack(rows)
    x[~torch.isfinite(x)] = 0
    x = x.to(dev)
    q = mx4_quantize(x)
    same_codes(q, x)
    assert torch.equal(mx4_dequantize(q).cpu(), values64(q).float())


def test_special_blocks(dev):
    x = torch.randn(4, 96, device=dev)
    x[0, 5], x[1, 40], x[2, 95] = math.nan, math.inf, -math.inf
    x[3, :32] = 0
    x[3, 33], x[3, 34] = -0.0, 1e-42
    q = mx4_quantize(x)
    same_codes(q, x)
    y = mx4_dequantize(q)
    bad = torch.zeros(4, 3, dtype=torch.bool, device=dev)
    bad[0, 0] = bad[1, 1] = bad[2, 2] = True
    assert torch.equal(y.unflatten(1, (3, 32)).isnan().all(-1), bad) and torch.equal(y.isnan().unflatten(1, (3, 32)).any(-1), bad)
    # every code under every scale
    codes = torch.arange(16, dtype=torch.uint8, device=dev).repeat(256, 1)
    q = MX4(codes, torch.arange(256, dtype=torch.uint8, device=dev)[:, None], 32)
    for dtype in TYPES:
        want = values64(q).to(dtype)
        assert torch.equal(mx4_dequantize(q, dtype=dtype).cpu().nan_to_num(777.0), want.nan_to_num(777.0))


def close(got, want, magnitude, terms):
    info = torch.finfo(got.dtype)
    bound = (info.eps / 2) * want.abs() + (terms + 1) * 2.0 ** -23 * magnitude + info.smallest_normal * info.eps / 2
    got = got.cpu().double()
    bad = ~((got - want).abs() <= bound * (1 + 2 ** -8))
    # beyond the middle between the type's largest value and the next step, which is max (1 + eps / 4), a value rounds to infinity
    bad &= ~(got.isinf() & (got.sign() == want.sign()) & (want.abs() + bound >= info.max * (1 + info.eps / 4)))
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, worst {float((got - want).abs()[bad].max())}"


def check(a, b, sizes=None, dtype=None):
    q = a if isinstance(a, MX4) else mx4_quantize(a)
    av, bv = values64(q), values64(b)
    T, N = av.shape[0], bv.shape[-2]
    s = None if sizes is None else torch.tensor(sizes, device=b.codes.device)
    c = mm_mx4(a, b, s, dtype=dtype)
    assert c.shape == (T, N) and c.dtype == (dtype or (torch.bfloat16 if isinstance(a, MX4) else a.dtype))
    want, size = torch.zeros(T, N, dtype=torch.float64), torch.zeros(T, N, dtype=torch.float64)
    r = 0
    for e, n in enumerate([T] if sizes is None else sizes):
        w = bv if sizes is None else bv[e]
        want[r:r + n], size[r:r + n] = av[r:r + n] @ w.T, av[r:r + n].abs() @ w.abs().T
        r += n
    close(c, want, size, a.length if isinstance(a, MX4) else a.shape[1])
    return c


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,N,K", [(1, 1, 1), (1, 130, 33), (3, 64, 256), (17, 200, 300), (40, 33, 64), (129, 257, 544), (300, 128, 1000), (600, 520, 288)])
def test_products(dev, T, N, K, dtype):
    a, w = torch.randn(T, K, device=dev).to(dtype), torch.randn(N, K, device=dev)
    b = mx4_quantize(w)
    c = check(a, b)
    assert torch.equal(mm_mx4(mx4_quantize(a), b, dtype=dtype), c)


@pytest.mark.parametrize("sizes,tail", [([1], 0), ([0, 1, 0], 0), ([5, 0, 130], 3), ([128, 128, 1], 0), ([0, 0], 4), ([2] * 70, 1), ([300, 31, 33], 0)], ids=str)
def test_grouped_products(dev, sizes, tail):
    for N, K, dtype in ((72, 96, torch.bfloat16), (136, 520, torch.float32), (33, 1000, torch.float16)):
        a = torch.randn(sum(sizes) + tail, K, device=dev).to(dtype)
        c = check(a, mx4_quantize(torch.randn(len(sizes), N, K, device=dev)), sizes)
        assert not c[sum(sizes):].any()


def test_scales_far_apart(dev):
    """Exponents over the whole range of the scale byte, where the product fits fp32."""
    T, N, K = 40, 48, 256
    g = torch.Generator().manual_seed(3)
    q = [MX4(torch.randint(0, 256, (n, K // 2), dtype=torch.uint8, generator=g).to(dev), torch.randint(lo, hi, (n, K // 32), generator=g).to(torch.uint8).to(dev), K)
         for n, lo, hi in ((T, 0, 120), (N, 135, 254))]
    check(q[0], q[1], dtype=torch.float32)
    check(q[1], q[0], dtype=torch.float32)


def test_views_and_nan(dev):
    a, w = torch.randn(20, 96, device=dev), torch.randn(50, 96, device=dev)
    b = mx4_quantize(w)
    want = mm_mx4(a, b)
    for off in (0, 1, 16):
        codes, scales = torch.zeros(50, 48 + 32, dtype=torch.uint8, device=dev), torch.zeros(50, 3 + 16, dtype=torch.uint8, device=dev)
        v = MX4(codes[:, off:off + 48].copy_(b.codes), scales[:, off:off + 3].copy_(b.scales), 96)
        assert torch.equal(mm_mx4(a, v), want) and torch.equal(mx4_dequantize(v), mx4_dequantize(b))
    assert torch.equal(mm_mx4(a.T.contiguous().T, b), want)
    assert torch.equal(mm_mx4(a, MX4(b.codes.T.contiguous().T, b.scales.T.contiguous().T, 96)), want)
    wide = torch.randn(20, 200, device=dev)
    assert torch.equal(mx4_quantize(wide[:, 3:99]).codes, mx4_quantize(wide[:, 3:99].contiguous()).codes)
    assert torch.equal(mx4_quantize(a[:1].expand(5, 96)).codes, mx4_quantize(a[:1]).codes.expand(5, -1))
    a[7, 50] = math.nan
    c = mm_mx4(a, b)
    assert c[7].isnan().all() and torch.equal(c[:7], want[:7]) and torch.equal(c[8:], want[8:])
    s = torch.tensor([7, 1, 12], device=dev)
    three = MX4(b.codes.repeat(3, 1, 1), b.scales.repeat(3, 1, 1), 96)
    three.scales[1] = 255
    c = mm_mx4(a, three, s)
    assert c[7].isnan().all() and torch.equal(c[:7], want[:7]) and torch.equal(c[8:], want[8:])


def test_empty_operands(dev):
    q = mx4_quantize(torch.empty(0, 40, device=dev))
    assert q.codes.shape == (0, 32) and mx4_dequantize(q).shape == (0, 40)
    b = mx4_quantize(torch.randn(6, 40, device=dev))
    assert mm_mx4(q, b).shape == (0, 6) and mm_mx4(b, q).shape == (6, 0)
    none = mx4_quantize(torch.empty(4, 0, device=dev))
    assert mx4_dequantize(none).shape == (4, 0) and not mm_mx4(none, none).any()


def test_graph_and_streams(dev):
    a, s = torch.randn(70, 160, device=dev, dtype=torch.bfloat16), torch.tensor([30, 0, 40], device=dev)
    b = mx4_quantize(torch.randn(3, 72, 160, device=dev))
    mm_mx4(a, b, s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mm_mx4(a, b, s)
    for sizes in ([30, 0, 40], [0, 70, 0], [10, 10, 10]):
        s.copy_(torch.tensor(sizes))
        a.normal_()
        eager = mm_mx4(a, b, s)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = mm_mx4(a, b, s)
    torch.cuda.synchronize()
    assert torch.equal(other, eager)


def test_refusals(dev):
    a, b = torch.randn(4, 64, device=dev), mx4_quantize(torch.randn(6, 64, device=dev))
    s = torch.tensor([4], device=dev)
    three = MX4(b.codes[None], b.scales[None], 64)
    for args in ((a[0], b), (a[:, :63], b), (a, three), (a, b, s), (a, three, torch.tensor([2, 2], device=dev)), (a, three, s.float()), (a, three, s.cpu()),
                 (a, MX4(b.codes[:, 1:], b.scales, 64)), (a, MX4(b.codes, b.scales[:5], 64)), (a, MX4(b.codes.int(), b.scales, 64))):
        with pytest.raises(AssertionError):
            mm_mx4(*args)
    for call in (lambda: mm_mx4(a.double(), b), lambda: mm_mx4(a, b, dtype=torch.float64), lambda: mx4_quantize(a.int()), lambda: mx4_dequantize(b, dtype=torch.int8)):
        with pytest.raises(NotImplementedError):
            call()
    with pytest.raises(RuntimeError, match="gradient"):
        mm_mx4(a.requires_grad_(), b)
    with torch.no_grad():
        mm_mx4(a, b)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tile", range(1, 5))
def test_every_tile(dev, tile, dtype):
    """Each tile on sizes that it would not be chosen for; values quantised within the call and before are the same bits."""
    for sizes, K, N, tail in (([3, 0, 5, 1], 64, 128, 2), ([33, 0, 64, 65, 31, 2], 130, 77, 11), ([300, 5], 2048, 264, 3), ([1] * 70, 40, 8, 0), ([150], 3000, 66, 0)):
        a = (torch.randn(sum(sizes) + tail, K, device=dev) * torch.exp(4 * torch.randn(sum(sizes) + tail, 1, device=dev))).to(dtype)
        b, s = mx4_quantize(torch.randn(len(sizes), N, K, device=dev)), torch.tensor(sizes, device=dev)
        c = mm_mx4(a, b, s, _tile=tile)
        q = mx4_quantize(a)
        again = mm_mx4(q, b, s, dtype=dtype, _tile=tile)
        # a row scaled beyond fp16's range holds infinities, which stand for NaN: rows of NaN on every side
        assert torch.equal(again.isnan(), c.isnan()) and torch.equal(again[~c.isnan()], c[~c.isnan()])
        av, bv = values64(q), values64(b)
        want, size = torch.zeros(c.shape, dtype=torch.float64), torch.zeros(c.shape, dtype=torch.float64)
        r = 0
        for e, n in enumerate(sizes):
            want[r:r + n], size[r:r + n] = av[r:r + n] @ bv[e].T, av[r:r + n].abs() @ bv[e].abs().T
            r += n
        assert torch.equal(want.isnan(), c.cpu().isnan()) and not want.isnan().all()
        fine = ~want.isnan()
        close(c.cpu()[fine], want[fine], size[fine], K)


@pytest.mark.parametrize("N", [40, 500, 3000, 6000])
def test_few_rows_over_many_columns(dev, N):
    """One or two rows under the widths at which a tile of few rows changes its columns; values and codes alike."""
    for K in (32, 128, 160, 2080, 2070):
        b = mx4_quantize(torch.randn(N, K, device=dev))
        for dtype in TYPES:
            a = torch.randn(2, K, device=dev).to(dtype)
            c = check(a, b)
            assert torch.equal(mm_mx4(mx4_quantize(a), b, dtype=dtype), c)


def test_rows_far_apart(dev):
    """Rows further apart than a tile's 31-bit offsets reach, of values and of codes."""
    far, K, N = (1 << 23) + 32, 96, 40
    a, b = torch.randn(3, K, device=dev).bfloat16(), mx4_quantize(torch.randn(N, K, device=dev))
    av = torch.empty(3, far, dtype=a.dtype, device=dev)[:, :K].copy_(a)
    q = mx4_quantize(a)
    qv = MX4(torch.empty(3, far, dtype=torch.uint8, device=dev)[:, :q.codes.shape[1]].copy_(q.codes), q.scales, K)
    for rows in (3, 1):
        want = mm_mx4(a[:rows], b)
        assert torch.equal(mm_mx4(av[:rows], b), want)
        assert torch.equal(mm_mx4(MX4(qv.codes[:rows], qv.scales[:rows], K), b), want)
    assert torch.equal(mx4_dequantize(qv), mx4_dequantize(q)) and torch.equal(mx4_quantize(av).codes, q.codes)


@pytest.mark.parametrize("sizes,N", [([300, 2, 500], 1500), ([300, 0, 1500, 700], 2000), ([900, 1100, 600, 700], 4000)])
def test_rounds_of_the_largest_tile(dev, sizes, N):
    """Last rounds in quarters, in halves and behind whole ones, under contractions that end at every step of the loop."""
    T = sum(sizes) + 5
    s = torch.tensor(sizes, device=dev)
    for K in (32, 128, 256, 384, 512, 640, 1056, 1312):
        a, b = mx4_quantize(torch.randn(T, K, device=dev)), mx4_quantize(torch.randn(len(sizes), N, K, device=dev))
        c = mm_mx4(a, b, s, _tile=4)
        av, bv = mx4_dequantize(a), mx4_dequantize(b)
        want, size, r = torch.zeros(T, N, dtype=torch.float64, device=dev), torch.zeros(T, N, dtype=torch.float64, device=dev), 0
        for e, n in enumerate(sizes):
            want[r:r + n] = av[r:r + n].double() @ bv[e].double().T
            size[r:r + n] = av[r:r + n].double().abs() @ bv[e].double().abs().T
            r += n
        close(c, want.cpu(), size.cpu(), K)
