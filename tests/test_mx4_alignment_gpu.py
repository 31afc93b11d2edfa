"""Codes and scales off the 16-byte boundaries, and sizes that do not fit, on every kernel of the 4-bit product."""

import math

import pytest
import torch

from triturus_amd.mx4 import MX4, mm_mx4, mx4_quantize

pytestmark = pytest.mark.gpu


def moved(q, by, gap):
    """The same rows `by` bytes off the boundaries, `gap` bytes of junk behind each; NaN's scale byte around the scales."""
    out = []
    for t, fill in ((q.codes, 0x77), (q.scales, 255)):
        width, rows = t.shape[-1], t[..., 0].numel()
        room = torch.full((rows * (width + gap) + by + 64,), fill, dtype=torch.uint8, device=t.device)
        view = room[by:by + rows * (width + gap)].view(*t.shape[:-1], width + gap)[..., :width]
        out.append(view.copy_(t))
    return MX4(*out, q.length)


@pytest.mark.parametrize("tile", range(0, 5))
@pytest.mark.parametrize("sizes,N,tail", [([3, 0, 5, 1], 33, 2), ([300, 5, 129], 264, 3), ([700, 0, 1100], 1500, 0)], ids=str)
def test_codes_at_any_address(dev, tile, sizes, N, tail):
    s = torch.tensor(sizes, dtype=torch.int32, device=dev)
    T, E = sum(sizes) + tail, len(sizes)
    for K in (32, 96, 128, 160, 256, 520, 1312):  # contractions that end at every step, rows of fewer than 4 blocks among them
        a, b = mx4_quantize(torch.randn(T, K, device=dev)), mx4_quantize(torch.randn(E, N, K, device=dev))
        for dtype in (torch.bfloat16, torch.float32):
            want = mm_mx4(a, b, s, dtype=dtype, _tile=tile)
            assert not want[T - tail:].any() and not want.isnan().any()
            for by, gap in ((1, 0), (4, 16), (16, 3), (7, 9), (0, 1)):
                where = (K, dtype, by, gap)
                assert torch.equal(mm_mx4(moved(a, by, gap), moved(b, by, gap), s, dtype=dtype, _tile=tile), want), where
            assert torch.equal(mm_mx4(a, moved(b, 5, 2), s, dtype=dtype, _tile=tile), want)
            assert torch.equal(mm_mx4(moved(a, 3, 1), b, s, dtype=dtype, _tile=tile), want)


@pytest.mark.parametrize("tile", range(0, 5))
@pytest.mark.parametrize("sizes", [[5, -3, 9, 4], [10, 1000, 7, 3], [1 << 30] * 4, [-1] * 4, [0, 0, 0, 300]], ids=str)
def test_sizes_that_do_not_fit_are_clamped(dev, sizes, tile):
    T, K, N = 300, 160, 72
    x = torch.randn(T, K, device=dev).bfloat16()
    b = mx4_quantize(torch.randn(4, N, K, device=dev))
    fit, left = [], T
    for n in sizes:
        fit.append(min(max(n, 0), left))
        left -= fit[-1]
    for a in (x, mx4_quantize(x)):
        for dtype in (torch.int32, torch.int64):
            got = mm_mx4(a, b, torch.tensor(sizes, dtype=dtype, device=dev), _tile=tile)
            assert torch.equal(got, mm_mx4(a, b, torch.tensor(fit, dtype=dtype, device=dev), _tile=tile))
            assert not got[T - left:].any()


@pytest.mark.parametrize("tile", range(0, 5))
def test_neighbours_do_not_leak(dev, tile):
    """NaN in other groups' rows, in other matrices and behind the last group stays there, on and off the boundaries."""
    sizes, N = [130, 0, 70, 300], 264
    s, T = torch.tensor(sizes, device=dev), 509
    for K in (40, 320):
        x = torch.randn(T, K, device=dev).bfloat16()
        b = mx4_quantize(torch.randn(4, N, K, device=dev))
        clean = mm_mx4(x, b, s, _tile=tile)
        x[130:200] = math.nan
        x[500:] = math.inf
        b.scales[1] = 255
        b.scales[2] = 255
        keep = torch.ones(T, dtype=torch.bool, device=dev)
        keep[130:200] = False
        for a in (x, mx4_quantize(x), moved(mx4_quantize(x), 3, 5)):
            for w in (b, moved(b, 3, 5)):
                c = mm_mx4(a, w, s, dtype=torch.bfloat16, _tile=tile)
                assert torch.equal(c[keep], clean[keep]) and c[130:200].isnan().all() and not c[500:].any()
